// Key/value caches held in 8 bits: writing, reading back, and attention over them (layout and definitions: mz_kv8 in
// mimizuku.h). Plain kernels: one wave per (row, head), or per query.
#include "mz_common.h"
#include "mz_kernels.h"

#include <algorithm>

namespace {

enum { I8 = 0, E4M3 = 1 };

// element of position t (of its block) and channel d in a block of values
__device__ __forceinline__ int v_at(int t, int d) { return ((d >> 1) * 4 + (t >> 3)) * 16 + (d & 1) * 8 + (t & 7); }

// what a code stands for, without its scale
template <int FMT>
__device__ __forceinline__ float code_value(unsigned char c) {
    if (FMT == I8) return (float)(signed char)c;
    const int e = (c >> 3) & 15, m = c & 7;
    if (e == 15 && m == 7) return NAN;
    return copysignf(e ? ldexpf(1.f + m * 0.125f, e - 7) : ldexpf((float)m, -9), c & 128 ? -1.f : 1.f);
}

// f16(f32(code * scale)). The product is kept from the compiler: it would fold it and the conversion into one mixed-width
// multiply-add of a positive zero, which rounds once and makes -0 to +0.
__device__ __forceinline__ f16 stands_for(float code, float scale) {
    float v = code * scale;
    asm("" : "+v"(v));
    return (f16)v;
}

// T x / top rounded as the real quotient would be. y = T x is exact in 32 bits (an fp16 value times 127 or 7 * 64), and
// the quotient of two such numbers is either halfway between two codes, and then a number of 32 bits, or at least 2^-19
// (relative) away from halfway; v is the quotient to the nearest 32-bit number (one correction of q by the exact
// remainder), so that rounding it again gives the code of the real quotient. rc = 1 / top.
template <int FMT>
__device__ __forceinline__ float quotient(float x, float top, float rc) {
    const float y = x * (FMT == I8 ? 127.f : 448.f), q = y * rc;
    return fmaf(fmaf(-q, top, y), rc, q);
}

// a block's scale and 1 / top from the largest magnitude's fp16 bits (NaN and infinities above every number's)
template <int FMT>
__device__ __forceinline__ void block_scale(unsigned bits, float& top, float& rc, float& scale) {
    top = (float)__builtin_bit_cast(f16, (unsigned short)bits);
    scale = bits < 0x7c00u ? top / (FMT == I8 ? 127.f : 448.f) : NAN;
    if (bits == 0 || bits >= 0x7c00u) top = rc = 0.f;  // codes 0
    else rc = 1.f / top;
}

template <int FMT>
__device__ __forceinline__ unsigned char code_of(f16 x, float top, float rc) {
    const float v = top > 0.f ? quotient<FMT>((float)x, top, rc) : 0.f;
    if (FMT == I8) return (unsigned char)(signed char)(int)rintf(v);
    return (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 255);
}

__device__ __forceinline__ unsigned magnitude(f16 x) { return __builtin_bit_cast(unsigned short, x) & 0x7fffu; }

// row r's slot and positions; false if there is nothing to do for it
struct Row {
    long slot;
    int p, n;
};
__device__ __forceinline__ bool row_of(const MzKv8& kv, const MzKv8Io& a, int r, Row& o) {
    o.slot = a.slot ? a.slot[r] : r;
    const long p = (long)a.pos_add + (a.pos ? a.pos[(long)r * a.pos_stride] : 0);
    o.n = a.count ? min(max(a.count[r], 0), a.tokens) : a.tokens;
    o.p = (int)p;
    return o.slot >= 0 && o.slot < kv.slots && p >= 0 && p <= (long)kv.blocks * MZ_KV_BLK;
}

template <int FMT>
__global__ void __launch_bounds__(64) write_kernel(MzKv8 kv, MzKv8Io a) {
    const int r = blockIdx.x / kv.heads, h = blockIdx.x - r * kv.heads, lane = threadIdx.x;
    Row w;
    if (!row_of(kv, a, r, w) || w.n <= 0 || w.p + (long)w.n > (long)kv.blocks * MZ_KV_BLK) return;
    if (a.slot)
        for (int i = r + 1; i < a.rows; i++)
            if (a.slot[i] == w.slot) return;
    const long sh = w.slot * kv.heads + h;
    const int open = kv.open[sh], first = w.p / MZ_KV_BLK, last = (w.p + w.n - 1) / MZ_KV_BLK;
    for (int side = 0; side < 2; side++) {
        const f16* src = (side ? a.v : a.k) + r * a.row_stride + h * a.head_stride;
        unsigned char* codes = (side ? kv.v : kv.k) + sh * kv.blocks * MZ_KV_TILE;
        float* scales = (side ? kv.v_scale : kv.k_scale) + sh * kv.blocks;
        f16* op = (side ? kv.v_open : kv.k_open) + sh * MZ_KV_TILE;
        auto at = [&](int t) { return side ? v_at(t, lane) : t * 64 + lane; };  // lane: the channel
        for (int b = first; b <= last; b++) {
            const int off = max(w.p - b * MZ_KV_BLK, 0), end = min(w.p + w.n - b * MZ_KV_BLK, MZ_KV_BLK);
            f16 x[MZ_KV_BLK];
            unsigned top = 0;
            for (int t = 0; t < end; t++) {
                if (t >= off) x[t] = src[(long)(b * MZ_KV_BLK + t - w.p) * a.token_stride + lane];
                else if (open == b + 1) x[t] = op[at(t)];
                else x[t] = stands_for(code_value<FMT>(codes[(long)b * MZ_KV_TILE + at(t)]), scales[b]);
                top = max(top, magnitude(x[t]));
            }
            if (end < MZ_KV_BLK) {
                for (int t = open == b + 1 ? off : 0; t < end; t++) op[at(t)] = x[t];
                continue;
            }
            float ft, rc, sc;
            block_scale<FMT>((unsigned)wave_max((float)top), ft, rc, sc);
            for (int t = 0; t < MZ_KV_BLK; t++) codes[(long)b * MZ_KV_TILE + at(t)] = code_of<FMT>(x[t], ft, rc);
            if (lane == 0) scales[b] = sc;
        }
    }
    if (lane == 0) kv.open[sh] = (w.p + w.n) % MZ_KV_BLK ? last + 1 : 0;
}

template <int FMT>
__global__ void __launch_bounds__(64) read_kernel(MzKv8 kv, MzKv8Io a) {
    const int r = blockIdx.x / kv.heads, h = blockIdx.x - r * kv.heads, lane = threadIdx.x;
    Row w;
    if (!row_of(kv, a, r, w)) return;
    const long sh = w.slot * kv.heads + h;
    const int open = kv.open[sh];
    for (int i = 0; i < w.n && w.p + i < kv.blocks * MZ_KV_BLK; i++) {
        const int b = (w.p + i) / MZ_KV_BLK, t = (w.p + i) % MZ_KV_BLK;
        const long o = r * a.row_stride + i * a.token_stride + h * a.head_stride + lane, e = (sh * kv.blocks + b) * MZ_KV_TILE;
        if (a.k)
            a.k[o] = open == b + 1 ? kv.k_open[sh * MZ_KV_TILE + t * 64 + lane]
                                   : stands_for(code_value<FMT>(kv.k[e + t * 64 + lane]), kv.k_scale[sh * kv.blocks + b]);
        if (a.v)
            a.v[o] = open == b + 1 ? kv.v_open[sh * MZ_KV_TILE + v_at(t, lane)]
                                   : stands_for(code_value<FMT>(kv.v[e + v_at(t, lane)]), kv.v_scale[sh * kv.blocks + b]);
    }
}

// ---------------------------------------------------------------- attention
//
// One pass over the cache with the running maximum and sum of the softmax. A workgroup takes 16 QT queries of one (row,
// cache head) (its tokens times the query heads that share the cache head) and a share of the blocks; its four waves
// take the blocks in turn, each with a state of its own, and join them at the end.
//
// Per block of 32 positions, with 16x16x32 products: S^T = K Q^T, the rows of tile j being positions 8 (i / 4) + 4 j + i % 4,
// so that lane (query c, group g) of the two results holds the eight positions 8 g .. 8 g + 7 of its query. These
// are, in this order, the k values of that lane in the product O^T = V^T P^T: the probabilities go from one product to the
// other in registers, with no exchange between lanes. The values are kept so that one 16-byte load gives a lane
// both channels 2 p and 2 p + 1 of its eight positions, the keys so that one gives 16 channels of a position.
//
// Codes become fp16 exactly, the products sum in 32 bits, the keys' scale goes into the exponent, the values' into
// the block's addition to the state. P is rounded to fp16 (half a step 2^-11 relative, as the output's own rounding); it is
// at most 2^8, because the maximum of a state is moved only when a score passes it by more than 8 (in powers of two): most
// blocks need no exchange between lanes and no rescaling.

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f, NOTHING = -1e30f;

// eight codes as fp16
template <int FMT>
__device__ __forceinline__ f16x8 widen(unsigned lo, unsigned hi) {
    f16x2 r[4];
    if (FMT == I8) {
        // the byte c + 128 under the high byte of 1024 is the number 1152 + c
        const unsigned x[2] = {lo ^ 0x80808080u, hi ^ 0x80808080u};
        const f16x2 bias = {(f16)1152.f, (f16)1152.f};
#pragma unroll
        for (int i = 0; i < 4; i++)
            r[i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x[i >> 1], i & 1 ? 0x04030402u : 0x04010400u)) - bias;
    } else {
        r[0] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
        r[1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
        r[2] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
        r[3] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
    }
    return f16x8{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
}

// maximum / sum over the four lanes of a column (lane ^ 16, ^ 32), in each of them
__device__ __forceinline__ float column_max(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return pair32_max(fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1])));
}
__device__ __forceinline__ float column_sum(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return pair32_sum(__builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]));
}

// what a row's queries see: token i positions first .. min(base + (causal ? i : 0), cap) - 1 of its slot
struct Seen {
    long slot, base;
    int cap, first, count;
    __device__ __forceinline__ int end(const MzKv8Attn& a, int i) const {
        return (int)min(max(base + (a.causal ? i : 0), 0L), (long)cap);
    }
};
__device__ __forceinline__ Seen seen_of(const MzKv8& kv, const MzKv8Attn& a, int r) {
    Seen s;
    s.slot = a.slot ? a.slot[r] : r;
    s.cap = kv.blocks * MZ_KV_BLK;
    s.base = (long)a.len_add + (a.len ? a.len[(long)r * a.len_stride] : 0);
    s.first = a.first ? max(a.first[r], 0) : 0;
    s.count = a.count ? min(max(a.count[r], 0), a.tokens) : a.tokens;
    if (s.slot < 0 || s.slot >= kv.slots) s.slot = s.cap = 0;
    return s;
}

// head h's row of alignment probabilities of (r, i), or null
__device__ __forceinline__ float* align_row(const MzKv8Attn& a, int r, int i, int h) {
    const int s = a.head_slot[h];
    if (s < 0 || s >= a.align_heads) return nullptr;
    for (int j = 0; j < h; j++)
        if (a.head_slot[j] == s) return nullptr;
    return a.align + (((long)r * a.tokens + i) * a.align_heads + s) * a.align_cols;
}

// scores (in powers of two) to probabilities, by all threads of the workgroup; 0 where nothing is seen
__device__ __forceinline__ void align_finish(float* row, int cols, int lo, int hi, float lse2) {
    for (int p = threadIdx.x; p < cols; p += 256)
        row[p] = p >= lo && p < hi ? __builtin_amdgcn_exp2f(row[p] - lse2) : 0.f;
}

struct Launch {
    int qt, tiles, splits;  // queries a workgroup / 16, such tiles of a (row, cache head), workgroups the blocks are shared by
};
constexpr int STATE = 66;  // floats of a query's partial state: 64 channels, maximum, sum

template <int FMT, int QT, bool ALIGN>
__global__ void __launch_bounds__(256) attn_kernel(MzKv8 kv, MzKv8Attn a, Launch n) {
    __shared__ float red[4][16][68], ms[4][16], ls[4][16];
    __shared__ float* als[16];
    __shared__ float lse2s[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    // workgroups of one (row, cache head) on one XCD (they share its keys and values where there are several tiles), the
    // tiles that see most first
    const unsigned per = 8u * n.tiles * n.splits, id = blockIdx.x, rem = id % per;
    const long pair = (long)(id / per) * 8 + (rem & 7);
    if (pair >= (long)a.rows * kv.heads) return;
    const int tile = n.tiles - 1 - (int)(rem >> 3) / n.splits, split = (int)(rem >> 3) % n.splits;
    const int r = (int)(pair / kv.heads), kh = (int)(pair - (long)r * kv.heads), grp = a.heads / kv.heads;
    const Seen s = seen_of(kv, a, r);
    const int q0 = tile * 16 * QT, nq = a.tokens * grp, qn = min(q0 + 16 * QT, nq);  // this tile's queries
    if (q0 / grp >= s.count) return;  // none of its tokens is there
    const int hi = s.end(a, min((qn - 1) / grp, s.count - 1)), lo_end = s.end(a, q0 / grp);
    const int b_lo = s.first / MZ_KV_BLK, nb = max((hi + MZ_KV_BLK - 1) / MZ_KV_BLK - b_lo, 0);
    const int share = (nb + n.splits - 1) / n.splits, b0 = b_lo + min(split * share, nb), b1 = b_lo + min((split + 1) * share, nb);

    const long sh = s.slot * kv.heads + kh;
    const int open = s.cap ? kv.open[sh] - 1 : -1;
    const unsigned char* kc = kv.k + sh * kv.blocks * MZ_KV_TILE;
    const unsigned char* vc = kv.v + sh * kv.blocks * MZ_KV_TILE;
    const float* ksc = kv.k_scale + sh * kv.blocks;
    const float* vsc = kv.v_scale + sh * kv.blocks;

    f16x8 qf[QT][2];
    int end[QT];
    float* al[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int x = q0 + 16 * t + c, i = x / grp, h = kh * grp + x - i * grp;
        const bool on = x < nq && i < s.count;
        const f16* q = a.q + r * a.q_row + (on ? i * a.q_token + h * a.q_head : 0) + 16 * g;
        qf[t][0] = on ? ld8(q) : f16x8{};
        qf[t][1] = on ? ld8(q + 8) : f16x8{};
        end[t] = on ? s.end(a, i) : 0;
        if (ALIGN) al[t] = on ? align_row(a, r, i, h) : nullptr;
    }

    // a block as it lies: codes in d[0 .. 3], or the open block's fp16
    struct Raw {
        uint4 d[8];
        float ks, vs;
    };
    const unsigned ktok = 8 * (c >> 2) + (c & 3);  // row c of key tile 0; tile 1 is 4 positions on
    auto fetch = [&](int b, Raw& w) {
        if (b == open) {
            const f16* ko = kv.k_open + sh * MZ_KV_TILE;
            const f16* vo = kv.v_open + sh * MZ_KV_TILE;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                w.d[j] = *(const uint4*)(ko + (ktok + 4 * (j >> 1)) * 64 + 16 * g + 8 * (j & 1));
                w.d[4 + j] = *(const uint4*)(vo + ((16 * (j >> 1) + c) * 4 + g) * 16 + 8 * (j & 1));
            }
            w.ks = w.vs = 1.f;
        } else {
            const unsigned char* k = kc + (long)b * MZ_KV_TILE;
            const unsigned char* v = vc + (long)b * MZ_KV_TILE;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                w.d[j] = *(const uint4*)(k + (ktok + 4 * j) * 64 + 16 * g);
                w.d[2 + j] = *(const uint4*)(v + ((16 * j + c) * 4 + g) * 16);
            }
            w.ks = ksc[b];
            w.vs = vsc[b];
        }
    };

    float m[QT], l[QT];
    f32x4 acc[QT][4];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        m[t] = NOTHING;
        l[t] = 0.f;
#pragma unroll
        for (int u = 0; u < 4; u++) acc[t][u] = f32x4{};
    }
    const float scale2 = a.scale * LOG2E;
    auto block = [&](int b, const Raw& w) {
        f16x8 kf[2][2], vf[4];
        const int p0 = b * MZ_KV_BLK + 8 * g;  // this lane's positions
        if (b == open) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                kf[j >> 1][j & 1] = __builtin_bit_cast(f16x8, w.d[j]);
                vf[j] = __builtin_bit_cast(f16x8, w.d[4 + j]);
#pragma unroll
                for (int e = 0; e < 8; e++)  // what no query of the tile sees may be no number
                    if (p0 + e < s.first || p0 + e >= hi) vf[j][e] = (f16)0.f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                kf[j][0] = widen<FMT>(w.d[j].x, w.d[j].y);
                kf[j][1] = widen<FMT>(w.d[j].z, w.d[j].w);
                vf[2 * j] = widen<FMT>(w.d[2 + j].x, w.d[2 + j].y);
                vf[2 * j + 1] = widen<FMT>(w.d[2 + j].z, w.d[2 + j].w);
            }
        }
        const float cs = scale2 * w.ks;
        const bool whole = b * MZ_KV_BLK >= s.first && (b + 1) * MZ_KV_BLK <= lo_end;  // seen by every query
#pragma unroll
        for (int t = 0; t < QT; t++) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const f32x4 d = mfma16(kf[j][1], qf[t][1], mfma16(kf[j][0], qf[t][0], f32x4{}));
#pragma unroll
                for (int e = 0; e < 4; e++) x[4 * j + e] = d[e] * cs;
            }
            if (!whole)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (p0 + e < s.first || p0 + e >= end[t]) x[e] = -INFINITY;
            if (ALIGN && al[t])
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (p0 + e >= s.first && p0 + e < min(end[t], a.align_cols)) al[t][p0 + e] = x[e];
            const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            if (__ballot(top > m[t] + 8.f)) {
                const float mn = fmaxf(m[t], column_max(top)), f = __builtin_amdgcn_exp2f(m[t] - mn);
                m[t] = mn;
                l[t] *= f;
#pragma unroll
                for (int u = 0; u < 4; u++) acc[t][u] *= f;
            }
            f16x8 p;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[e] = __builtin_amdgcn_exp2f(x[e] - m[t]);
                p[e] = (f16)x[e];
            }
            l[t] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
            const bool any = whole || b * MZ_KV_BLK < end[t];  // (0 times a scale or a value that is no number is none)
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const f32x4 d = mfma16(vf[u], p, f32x4{});
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y = fmaf(d[e], w.vs, acc[t][u][e]);
                    acc[t][u][e] = whole || any ? y : acc[t][u][e];
                }
            }
        }
    };
    Raw w0, w1;
    int b = b0 + wave;
    if (b < b1) fetch(b, w0);
    for (; b < b1; b += 8) {
        if (b + 4 < b1) fetch(b + 4, w1);
        block(b, w0);
        if (b + 4 < b1) {
            if (b + 8 < b1) fetch(b + 8, w0);
            block(b + 4, w1);
        }
    }

    // the four waves' states joined, 16 queries at a time; accumulator u of lane (c, g) holds channels
    // 32 (u / 2) + 8 g + 2 e + u % 2 of query c
    const int col = tid >> 4, d4 = (tid & 15) * 4;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const float lt = column_sum(l[t]);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float* o = &red[wave][c][32 * u + 8 * g];
            *(f32x4*)o = f32x4{acc[t][2 * u][0], acc[t][2 * u + 1][0], acc[t][2 * u][1], acc[t][2 * u + 1][1]};
            *(f32x4*)(o + 4) = f32x4{acc[t][2 * u][2], acc[t][2 * u + 1][2], acc[t][2 * u][3], acc[t][2 * u + 1][3]};
        }
        if (g == 0) {
            ms[wave][c] = m[t];
            ls[wave][c] = lt;
            if (ALIGN && wave == 0) als[c] = al[t];
        }
        __syncthreads();
        const int x = q0 + 16 * t + col, i = x / grp, h = kh * grp + x - i * grp;
        const bool on = x < nq && i < s.count;
        float mm = fmaxf(fmaxf(ms[0][col], ms[1][col]), fmaxf(ms[2][col], ms[3][col])), ll = 0.f;
        f32x4 o = {};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float f = __builtin_amdgcn_exp2f(ms[k][col] - mm);
            ll = fmaf(f, ls[k][col], ll);
            const f32x4 y = *(const f32x4*)&red[k][col][d4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(f, y[e], o[e]);
        }
        if (n.splits > 1) {
            float* w = a.work + (((pair * n.tiles + tile) * n.splits + split) * (16 * QT) + 16 * t + col) * STATE;
            *(float2*)(w + d4) = float2{o[0], o[1]};
            *(float2*)(w + d4 + 2) = float2{o[2], o[3]};
            if (d4 == 0) *(float2*)(w + 64) = float2{mm, ll};
        } else {
            const float inv = ll == 0.f ? 0.f : 1.f / ll, lse2 = ll == 0.f ? -INFINITY : mm + __builtin_amdgcn_logf(ll);
            if (on) {
                st4(a.out + r * a.out_row + i * a.out_token + h * a.out_head + d4, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
                if (a.lse && d4 == 0) a.lse[((long)r * a.tokens + i) * a.heads + h] = lse2 * LN2;
            }
            if (ALIGN) {
                if (d4 == 0) lse2s[col] = lse2;
                __syncthreads();
                for (int k = 0; k < 16; k++)
                    if (als[k]) align_finish(als[k], a.align_cols, s.first, s.end(a, (q0 + 16 * t + k) / grp), lse2s[k]);
            }
        }
        __syncthreads();
    }
}

// The states of a query's splits joined, a workgroup a query: wave w takes splits w, w + 4, ...
__global__ void __launch_bounds__(256) attn_join_kernel(MzKv8 kv, MzKv8Attn a, Launch n) {
    __shared__ float red[4][64], ms[4], ls[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, grp = a.heads / kv.heads;
    const long id = blockIdx.x, ri = id / a.heads;
    const int h = (int)(id - ri * a.heads), r = (int)(ri / a.tokens), i = (int)(ri - (long)r * a.tokens);
    const Seen s = seen_of(kv, a, r);
    if (i >= s.count) return;
    const int x = i * grp + h % grp, qs = 16 * n.qt, tile = x / qs;
    const long pair = (long)r * kv.heads + h / grp;
    const float* w = a.work + ((pair * n.tiles + tile) * n.splits * qs + x - tile * qs) * STATE;
    float m = NOTHING, l = 0.f, o = 0.f;
    for (int k = wave; k < n.splits; k += 4) {
        const float* p = w + (long)k * qs * STATE;
        const float mk = p[64], lk = p[65], ok = p[lane], mn = fmaxf(m, mk);
        const float f = __builtin_amdgcn_exp2f(m - mn), fk = __builtin_amdgcn_exp2f(mk - mn);
        l = fmaf(l, f, lk * fk);
        o = fmaf(o, f, ok * fk);
        m = mn;
    }
    red[wave][lane] = o;
    if (lane == 0) {
        ms[wave] = m;
        ls[wave] = l;
    }
    __syncthreads();
    const float mm = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    l = o = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float f = __builtin_amdgcn_exp2f(ms[k] - mm);
        l = fmaf(f, ls[k], l);
        o = fmaf(f, red[k][lane], o);
    }
    const float lse2 = l == 0.f ? -INFINITY : mm + __builtin_amdgcn_logf(l);
    if (wave == 0) {
        a.out[r * a.out_row + i * a.out_token + h * a.out_head + lane] = (f16)(l == 0.f ? 0.f : o / l);
        if (a.lse && lane == 0) a.lse[((long)r * a.tokens + i) * a.heads + h] = lse2 * LN2;
    }
    if (a.head_slot)
        if (float* row = align_row(a, r, i, h)) align_finish(row, a.align_cols, s.first, s.end(a, i), lse2);
}

Launch attn_shape(const MzKv8& kv, const MzKv8Attn& a) {
    const long nq = (long)a.tokens * (a.heads / kv.heads), pairs = (long)a.rows * kv.heads;
    Launch n;
    n.qt = nq <= 16 ? 1 : nq <= 32 ? 2 : 4;
    n.tiles = (int)((nq + 16 * n.qt - 1) / (16 * n.qt));
    const long want = 2L * mz_cu_count() / (pairs * n.tiles);
    n.splits = (int)std::max(1L, std::min(want, (long)kv.blocks / 4));
    return n;
}

template <int FMT, bool ALIGN>
void attn_launch(hipStream_t s, const MzKv8& kv, const MzKv8Attn& a, const Launch& n, long grid) {
    if (n.qt == 1) hipLaunchKernelGGL((attn_kernel<FMT, 1, ALIGN>), dim3(grid), dim3(256), 0, s, kv, a, n);
    else if (n.qt == 2) hipLaunchKernelGGL((attn_kernel<FMT, 2, ALIGN>), dim3(grid), dim3(256), 0, s, kv, a, n);
    else hipLaunchKernelGGL((attn_kernel<FMT, 4, ALIGN>), dim3(grid), dim3(256), 0, s, kv, a, n);
}

}  // namespace

long mz_kv8_write_grid(const MzKv8& kv, const MzKv8Io& a) { return (long)a.rows * kv.heads; }
long mz_kv8_read_grid(const MzKv8& kv, const MzKv8Io& a) { return (long)a.rows * kv.heads; }

long mz_kv8_attn_grid(const MzKv8& kv, const MzKv8Attn& a) {
    const Launch n = attn_shape(kv, a);
    const long main = ((long)a.rows * kv.heads + 7) / 8 * 8 * n.tiles * n.splits, join = (long)a.rows * a.tokens * a.heads;
    return n.splits > 1 ? std::max(main, join) : main;
}

size_t mz_kv8_attn_work(const MzKv8& kv, const MzKv8Attn& a) {
    const Launch n = attn_shape(kv, a);
    return n.splits > 1 ? (size_t)a.rows * kv.heads * n.tiles * n.splits * 16 * n.qt * STATE * 4 : 0;
}

hipError_t mz_kv8_write_launch(hipStream_t s, const MzKv8& kv, const MzKv8Io& a) {
    const dim3 grid(mz_kv8_write_grid(kv, a));
    if (kv.format == I8) hipLaunchKernelGGL(write_kernel<I8>, grid, dim3(64), 0, s, kv, a);
    else hipLaunchKernelGGL(write_kernel<E4M3>, grid, dim3(64), 0, s, kv, a);
    return hipGetLastError();
}

hipError_t mz_kv8_read_launch(hipStream_t s, const MzKv8& kv, const MzKv8Io& a) {
    const dim3 grid(mz_kv8_read_grid(kv, a));
    if (kv.format == I8) hipLaunchKernelGGL(read_kernel<I8>, grid, dim3(64), 0, s, kv, a);
    else hipLaunchKernelGGL(read_kernel<E4M3>, grid, dim3(64), 0, s, kv, a);
    return hipGetLastError();
}

hipError_t mz_kv8_attn_launch(hipStream_t s, const MzKv8& kv, const MzKv8Attn& a) {
    const Launch n = attn_shape(kv, a);
    const long grid = ((long)a.rows * kv.heads + 7) / 8 * 8 * n.tiles * n.splits;
    if (kv.format == I8) a.align ? attn_launch<I8, true>(s, kv, a, n, grid) : attn_launch<I8, false>(s, kv, a, n, grid);
    else a.align ? attn_launch<E4M3, true>(s, kv, a, n, grid) : attn_launch<E4M3, false>(s, kv, a, n, grid);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || n.splits == 1) return e;
    hipLaunchKernelGGL(attn_join_kernel, dim3((long)a.rows * a.tokens * a.heads), dim3(256), 0, s, kv, a, n);
    return hipGetLastError();
}
