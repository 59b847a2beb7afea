// Key/value caches held in 8 bits: writing, reading back, and attention over them (layout and definitions: mz_kv8 in
// mimizuku.h).
#include "mz_common.h"
#include "mz_kernels.h"

#include <algorithm>
#include <type_traits>

namespace {

enum { I8 = 0, E4M3 = 1 };
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// element of position t (of its block) and channel d in a block of values
__device__ __forceinline__ int v_at(int t, int d) { return ((d >> 1) * 4 + (t >> 3)) * 16 + (d & 1) * 8 + (t & 7); }

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

// eight codes as bf16, whose 8 bits hold every code of either format
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
template <int FMT>
__device__ __forceinline__ bf16x8 widen_bf16(unsigned lo, unsigned hi) {
    u32x4 r;
    if (FMT == I8) {
#pragma unroll
        for (int i = 0; i < 4; i++) {  // (the high halves of two 32-bit numbers)
            const unsigned w = (i & 2 ? hi : lo) >> (i & 1) * 16;
            const float a = (float)(signed char)w, b = (float)(signed char)(w >> 8);
            r[i] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u);
        }
    } else {
        r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
        r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
        r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
        r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
    }
    return __builtin_bit_cast(bf16x8, r);
}

// a pair of fp16 numbers of eight bits as bf16
__device__ __forceinline__ unsigned as_bf16(f16x2 v) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, (float)v[1]), __builtin_bit_cast(unsigned, (float)v[0]), 0x07060302u);
}

// f16(f32(code * scale)). The product is kept from the compiler: it would fold it and the conversion into one mixed-width
// multiply-add of a positive zero, which rounds once and makes -0 to +0.
__device__ __forceinline__ f16 stands_for(f16 code, float scale) {
    float v = (float)code * scale;
    asm("" : "+v"(v));
    return (f16)v;
}
__device__ __forceinline__ f16x8 stand_for(f16x8 code, float scale) {
    f16x8 r;
#pragma unroll
    for (int e = 0; e < 8; e++) r[e] = stands_for(code[e], scale);
    return r;
}

// T x / top rounded as the real quotient would be. y = T x is exact in 32 bits (an fp16 value times 127 or 7 * 64), and
// the quotient of two such numbers is either halfway between two codes, and then a number of 32 bits, or at least 2^-19
// (relative) away from halfway; v is the quotient to the nearest 32-bit number (one correction of q by the exact
// remainder), so that rounding it again gives the code of the real quotient. rc = 1 / top.
template <int FMT>
__device__ __forceinline__ float quotient(f16 x, float top, float rc) {
    const float y = (float)x * (FMT == I8 ? 127.f : 448.f), q = y * rc;
    return fmaf(fmaf(-q, top, y), rc, q);
}

// four codes in a word. Whole numbers: adding 1.5 * 2^23 rounds to one, halves to even, and leaves it in the low byte.
template <int FMT>
__device__ __forceinline__ unsigned codes4(f16 a, f16 b, f16 c, f16 d, float top, float rc) {
    const float x[4] = {quotient<FMT>(a, top, rc), quotient<FMT>(b, top, rc), quotient<FMT>(c, top, rc), quotient<FMT>(d, top, rc)};
    if (FMT == I8) {
        unsigned u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = __builtin_bit_cast(unsigned, x[i] + 12582912.f);
        const unsigned lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
        return lo | hi;
    }
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], r, true);
}

// the larger magnitudes of two pairs of fp16 numbers as bits (NaN above infinity above every number)
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 larger(u16x2 m, unsigned pair) {
    return __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, pair & 0x7fff7fffu));
}

// a block's top, 1 / top (both 0 where all codes are 0) and scale, from every lane's largest magnitudes
template <int FMT>
__device__ __forceinline__ float block_scale(u16x2 m, float& top, float& rc) {
    const unsigned bits = (unsigned)wave_max((float)max(m[0], m[1]));
    top = rc = 0.f;
    if (bits >= 0x7c00u) return NAN;
    if (bits == 0) return 0.f;
    top = (float)__builtin_bit_cast(f16, (unsigned short)bits);
    rc = 1.f / top;
    return top / (FMT == I8 ? 127.f : 448.f);
}

// row r's slot and tokens i0 .. i0 + n - 1, the first of them at position p, without those before the cache; false if there is
// nothing to do for it
struct Row {
    long slot;
    int p, n, i0;
};
__device__ __forceinline__ bool row_of(const MzKv8& kv, const MzKv8Io& a, int r, Row& o) {
    // (if any array is there all are read, an absent one's place being some other word: the loads go out together)
    int slot = 0, pos = 0, count = 0;
    if (a.slot || a.pos || a.count) {
        slot = *(a.slot ? a.slot + r : kv.open);
        pos = *(a.pos ? a.pos + (long)r * a.pos_stride : kv.open);
        count = *(a.count ? a.count + r : kv.open);
    }
    o.slot = a.slot ? slot : r;
    const long p = (long)a.pos_add + (a.pos ? pos : 0);
    o.n = a.count ? min(max(count, 0), a.tokens) : a.tokens;
    o.i0 = (int)min(max(-p, 0L), (long)o.n);
    o.n -= o.i0;
    o.p = (int)max(p, 0L);
    return o.n > 0 && o.slot >= 0 && o.slot < kv.slots && p < (long)kv.blocks * MZ_KV_BLK;
}

// the same for a write, whose positions are all in the cache or not written
__device__ __forceinline__ bool write_row(const MzKv8& kv, const MzKv8Io& a, int r, Row& o) {
    return row_of(kv, a, r, o) && o.i0 == 0 && o.p + (long)o.n <= (long)kv.blocks * MZ_KV_BLK;
}

// Lanes over a block, keys: 8 channels of positions lane / 8 + 8 i; values: 4 channels of 8 positions, so that whole
// 16-byte pieces of the order of v are a lane's own.
//
// A wave codes one side of one block: its positions below `off` were there before (in the open block if `open`, else as
// codes), those below `end` are new. Positions that only stay in an open block are not touched.
template <int FMT>
struct Writer {
    const MzKv8& kv;
    const MzKv8Io& a;
    long sh;
    const f16* src;  // row, head and side applied
    int side, lane, p, n, open;

    int off, end;
    bool full, old;  // the block is whole now; its earlier positions are wanted
    f16x8 x[4] = {};  // keys: position lane / 8 + 8 i; values: channel 4 c + i, positions 8 g .. 8 g + 7

    // a block all of whose positions are new
    __device__ __forceinline__ void fetch(int b, u32x4 (&raw)[4]) const {
        const f16* s = src + (long)(b * MZ_KV_BLK - p) * a.token_stride;
        if (side == 0)
#pragma unroll
            for (int i = 0; i < 4; i++)
                raw[i] = __builtin_nontemporal_load((const u32x4*)(s + ((lane >> 3) + 8 * i) * a.token_stride + (lane & 7) * 8));
        else
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const u32x2 y = __builtin_nontemporal_load((const u32x2*)(s + ((lane >> 4) * 8 + j) * a.token_stride + (lane & 15) * 4));
                raw[j >> 1][(j & 1) * 2] = y[0];
                raw[j >> 1][(j & 1) * 2 + 1] = y[1];
            }
    }
    __device__ __forceinline__ void take(const u32x4 (&raw)[4]) {
        if (side == 0)
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = __builtin_bit_cast(f16x8, raw[i]);
        else
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const f16x4 y = __builtin_bit_cast(f16x4, u32x2{raw[j >> 1][(j & 1) * 2], raw[j >> 1][(j & 1) * 2 + 1]});
#pragma unroll
                for (int e = 0; e < 4; e++) x[e][j] = y[e];
            }
    }

    __device__ __forceinline__ void load(int b) {
        off = max(p - b * MZ_KV_BLK, 0);
        end = min(p + n - b * MZ_KV_BLK, MZ_KV_BLK);
        full = end == MZ_KV_BLK;
        const f16* s = src + (long)(b * MZ_KV_BLK - p) * a.token_stride;
        const long blk = sh * kv.blocks + b;
        if (side == 0) {
            const int d = (lane & 7) * 8;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = (lane >> 3) + 8 * i;
                x[i] = f16x8{};
                if (t >= off && t < end) x[i] = __builtin_nontemporal_load((const f16x8*)(s + t * a.token_stride + d));
            }
            old = off > 0 && (full || open != b);  // (the new ones are on their way before it is known which block is open)
            if (old)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = (lane >> 3) + 8 * i;
                    if (t >= off) continue;
                    if (open == b) x[i] = ld8(kv.k_open + sh * MZ_KV_TILE + t * 64 + d);
                    else {
                        const uint2 c = *(const uint2*)(kv.k + blk * MZ_KV_TILE + t * 64 + d);
                        x[i] = stand_for(widen<FMT>(c.x, c.y), kv.k_scale[blk]);
                    }
                }
        } else {
            const int d = (lane & 15) * 4, t0 = (lane >> 4) * 8;
            f16x4 y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int t = t0 + j;
                y[j] = f16x4{};
                if (t >= off && t < end) y[j] = __builtin_nontemporal_load((const f16x4*)(s + t * a.token_stride + d));
            }
            old = off > 0 && (full || open != b);
            if (old) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int at = ((lane & 15) * 2 + e) * 64 + (lane >> 4) * 16;
                    if (open == b) {
                        x[2 * e] = ld8(kv.v_open + sh * MZ_KV_TILE + at);
                        x[2 * e + 1] = ld8(kv.v_open + sh * MZ_KV_TILE + at + 8);
                    } else {
                        const uint4 u = *(const uint4*)(kv.v + blk * MZ_KV_TILE + at);
                        x[2 * e] = stand_for(widen<FMT>(u.x, u.y), kv.v_scale[blk]);
                        x[2 * e + 1] = stand_for(widen<FMT>(u.z, u.w), kv.v_scale[blk]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[e][j] = t0 + j < off ? x[e][j] : y[j][e];
        }
    }

    __device__ __forceinline__ void code(int b) const {
        const long blk = sh * kv.blocks + b;
        u16x2 m = {};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint4 u = __builtin_bit_cast(uint4, x[i]);
            m = larger(larger(larger(larger(m, u.x), u.y), u.z), u.w);
        }
        float top, rc;
        const float scale = block_scale<FMT>(m, top, rc);
        uint2 c[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[i] = uint2{codes4<FMT>(x[i][0], x[i][1], x[i][2], x[i][3], top, rc), codes4<FMT>(x[i][4], x[i][5], x[i][6], x[i][7], top, rc)};
            if (top == 0.f) c[i] = uint2{0, 0};
        }
        if (side == 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) *(uint2*)(kv.k + blk * MZ_KV_TILE + lane * 8 + 512 * i) = c[i];
            if (lane == 0) kv.k_scale[blk] = scale;
        } else {
            unsigned char* v = kv.v + blk * MZ_KV_TILE + (lane & 15) * 128 + (lane >> 4) * 16;
            *(uint4*)v = uint4{c[0].x, c[0].y, c[1].x, c[1].y};
            *(uint4*)(v + 64) = uint4{c[2].x, c[2].y, c[3].x, c[3].y};
            if (lane == 0) kv.v_scale[blk] = scale;
        }
    }

    __device__ __forceinline__ void store(int b) const {
        if (full) {
            code(b);
            return;
        }
        const int lo = old ? 0 : off;
        if (side == 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = (lane >> 3) + 8 * i;
                if (t >= lo && t < end) *(f16x8*)(kv.k_open + sh * MZ_KV_TILE + t * 64 + (lane & 7) * 8) = x[i];
            }
        } else {
            const int d = (lane & 15) * 4, t0 = (lane >> 4) * 8;
            f16* v = kv.v_open + sh * MZ_KV_TILE;
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (t0 + j >= lo && t0 + j < end)
#pragma unroll
                    for (int e = 0; e < 4; e++) v[v_at(t0 + j, d + e)] = x[e][j];
        }
    }
};

// 8 x 1500 positions of 20 heads (92 MB in and out) 19.8 us, 4.7 TB/s: a copy would take 14 behind the launch and the first round
// trips; the quotients' correction is 0.8. One position of 32 rows 5.0 us, a chain of four loads.
//
// Workgroup 0 of a (row, head) takes its first and its last block, which may want the open block and may leave one: a wave
// for the keys and one for the values of each. The others take the blocks between, 2 * per each, whose positions are all new:
// every wave `per` of keys or of values, the next one's on their way while one is coded.
template <int FMT>
__global__ void __launch_bounds__(256) write_kernel(MzKv8 kv, MzKv8Io a, int per) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), grp = blockIdx.x;
    const int r = blockIdx.z, h = blockIdx.y;
    Row w;
    if (!write_row(kv, a, r, w)) return;
    const int first = w.p / MZ_KV_BLK, last = (w.p + w.n - 1) / MZ_KV_BLK;
    if (grp && first + 1 + 2 * per * (grp - 1) >= last) return;
    if (a.slot)  // of rows that write to a slot the last one does
        for (int i = r + 1; i < a.rows; i += 64) {
            bool later = i + lane < a.rows && a.slot[i + lane < a.rows ? i + lane : i] == w.slot;
            if (__ballot(later)) {
                Row o;
                later = later && write_row(kv, a, i + lane, o);
                if (__ballot(later)) return;
            }
        }
    const long sh = w.slot * kv.heads + h;
    const int side = wave & 1;
    Writer<FMT> x{kv, a, sh, (side ? a.v : a.k) + r * a.row_stride + h * a.head_stride, side, lane, w.p, w.n, grp ? -1 : kv.open[sh] - 1};
    if (grp) {
        const int end = min(first + 1 + 2 * per * grp, last);
        int b = first + 1 + 2 * per * (grp - 1) + (wave >> 1);
        u32x4 raw[4];
        if (b < end) x.fetch(b, raw);
        for (; b < end; b += 2) {
            x.take(raw);
            if (b + 2 < end) x.fetch(b + 2, raw);
            x.code(b);
        }
        return;
    }
    const int b = wave < 2 ? first : last;
    const bool mine = wave < 2 || last > first;
    if (mine) x.load(b);
    __syncthreads();  // the open block is read before it is written
    if (mine) x.store(b);
    if (threadIdx.x == 0) kv.open[sh] = (w.p + w.n) % MZ_KV_BLK ? last + 1 : 0;
}

// a workgroup: keys and values of two blocks of a (row, head), a wave each (8 x 1500 positions of 20 heads, 92 MB in and out,
// 16.4 us, 5.6 TB/s; a copy reaches 6.6)
template <int FMT>
__global__ void __launch_bounds__(256) read_kernel(MzKv8 kv, MzKv8Io a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), side = wave & 1;
    const int r = blockIdx.z, h = blockIdx.y;
    f16* const base = side ? a.v : a.k;
    if (!base) return;
    Row w;
    if (!row_of(kv, a, r, w)) return;
    const int b = w.p / MZ_KV_BLK + (int)blockIdx.x * 2 + (wave >> 1);
    const int lo = max(w.p - b * MZ_KV_BLK, 0), hi = min((int)min((long)w.p + w.n, (long)kv.blocks * MZ_KV_BLK) - b * MZ_KV_BLK, MZ_KV_BLK);
    if (hi <= lo) return;
    const long sh = w.slot * kv.heads + h, blk = sh * kv.blocks + b;
    const bool open = kv.open[sh] == b + 1;
    f16* o = base + r * a.row_stride + h * a.head_stride + (b * MZ_KV_BLK - w.p + (long)w.i0) * a.token_stride;
    if (side == 0) {
        const int d = (lane & 7) * 8;
        f16x8 x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = (lane >> 3) + 8 * i;
            if (open) x[i] = ld8(kv.k_open + sh * MZ_KV_TILE + t * 64 + d);
            else {
                const uint2 c = *(const uint2*)(kv.k + blk * MZ_KV_TILE + t * 64 + d);
                x[i] = stand_for(widen<FMT>(c.x, c.y), kv.k_scale[blk]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = (lane >> 3) + 8 * i;
            if (t >= lo && t < hi) *(f16x8*)(o + t * a.token_stride + d) = x[i];
        }
    } else {
        const int c = lane & 15, g = lane >> 4;
        f16x8 x[4];  // channel 4 c + i, positions 8 g ..
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int at = ((2 * c + e) * 4 + g) * 16;
            if (open) {
                x[2 * e] = ld8(kv.v_open + sh * MZ_KV_TILE + at);
                x[2 * e + 1] = ld8(kv.v_open + sh * MZ_KV_TILE + at + 8);
            } else {
                const uint4 u = *(const uint4*)(kv.v + blk * MZ_KV_TILE + at);
                const float s = kv.v_scale[blk];
                x[2 * e] = stand_for(widen<FMT>(u.x, u.y), s);
                x[2 * e + 1] = stand_for(widen<FMT>(u.z, u.w), s);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int t = 8 * g + j;
            if (t >= lo && t < hi) *(f16x4*)(o + t * a.token_stride + 4 * c) = f16x4{x[0][j], x[1][j], x[2][j], x[3][j]};
        }
    }
}

// the most blocks that a row's positions can lie in
long spanned(const MzKv8& kv, const MzKv8Io& a) { return std::min(((long)a.tokens + MZ_KV_BLK - 2) / MZ_KV_BLK + 1, (long)kv.blocks); }
// Blocks between the first and the last that a wave takes (write_kernel): two where that leaves every CU four workgroups (8 x
// 1500 positions of 20 heads 19.8 us, 25.8 with one, 22.0 with four; 32 x 224 positions 15.6 / 22.5 / 16.2; but 1500 positions
// of one row 6.8 / 6.5 / 8.3).
int write_per(const MzKv8& kv, const MzKv8Io& a) {
    return (long)a.rows * kv.heads * std::max(0L, spanned(kv, a) - 2) >= 16L * mz_cu_count() ? 2 : 1;
}
long write_groups(const MzKv8& kv, const MzKv8Io& a, int per) { return 1 + (std::max(0L, spanned(kv, a) - 2) + 2 * per - 1) / (2 * per); }

// ---------------------------------------------------------------- attention
//
// One pass over the cache with the running maximum and sum of the softmax. A workgroup takes 16 QT queries of one (row,
// cache head) (its tokens times the query heads that share the cache head) and a share of the blocks; its waves take the
// blocks in turn, each with a state of its own, and join them at the end.
//
// Bound by memory for single tokens: 4,104 bytes a block, of which 32 rows x 20 heads x 1500 positions (126 MB) take 23.6 us,
// 6.7 TB/s behind the ~5 us of the launch and of the round trips to the first key and from the last (25.5 with six alignment
// heads). One row: those round trips, 7.6 us (8.7). Prompts: 8 of 224 tokens over up to 374 positions 13.2 us, the chain of the
// longest, 12 blocks one after the other, each with a barrier, a round trip through LDS and two products that wait for each
// other (waves wait half of their time, the vector units are busy for 39% of a CU's); over 1500 positions 39.4, vector
// instructions: about 150 a block of 16 queries, products included.
//
// Per block of 32 positions, with 16x16x32 products: S^T = K Q^T, the rows of tile j being positions 8 (i / 4) + 4 j + i % 4,
// so that lane (query c, group g) of the two results holds the eight positions 8 g .. 8 g + 7 of its query. These
// are, in this order, the k values of that lane in the product O^T = V^T P^T: the probabilities go from one product to the
// other in registers, with no exchange between lanes. The values are kept so that one 16-byte load gives a lane
// both channels 2 p and 2 p + 1 of its eight positions, the keys so that one gives 16 channels of a position.
//
// Codes become numbers of 16 bits exactly, the products sum in 32 bits, the keys' scale goes into the exponent, the values'
// into P. P goes into its product as the sum of two bf16 numbers: 16 bits (each rounding is at most 2^-8 of what it rounds),
// so that the error is the output's own rounding, and of the range of 32 bits, so that many positions far below a row's
// largest keep their share (two fp16 numbers end at 2^-24). The maximum of a state is moved only when a score passes it by more
// than 8 (in powers of two), so that most blocks need no exchange between lanes and no rescaling.

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f, NOTHING = -1e30f;

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

// v p for p = high + low
__device__ __forceinline__ f32x4 weighted(bf16x8 v, bf16x8 high, bf16x8 low, f32x4 to) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, high, __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, low, to, 0, 0, 0), 0, 0, 0);
}

__device__ __forceinline__ float lane_value(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// (the median of two numbers and infinity is the larger one. A maximum would make each operand quiet first, and so would a
// median with an infinity that the compiler knows.)
__device__ __forceinline__ float larger(float a, float b, float inf) { return __builtin_amdgcn_fmed3f(a, b, inf); }

// what a row's queries see: token i positions first .. min(base + (causal ? i : 0), cap) - 1 of its slot
struct Seen {
    long slot, base;
    int cap, first, count;
    __device__ __forceinline__ int end(const MzKv8Attn& a, int i) const {
        return (int)min(max(base + (a.causal ? i : 0), 0L), (long)cap);
    }
};
__device__ __forceinline__ Seen seen_of(const MzKv8& kv, const MzKv8Attn& a, int r) {
    // (if any array is there all are read, an absent one's place being some other word: the loads go out together, where
    // a branch around each would wait for one after the other)
    int slot = 0, first = 0, len = 0, count = 0;
    if (a.slot || a.first || a.len || a.count) {
        slot = *(a.slot ? a.slot + r : kv.open);
        first = *(a.first ? a.first + r : kv.open);
        len = *(a.len ? a.len + (long)r * a.len_stride : kv.open);
        count = *(a.count ? a.count + r : kv.open);
        slot = __builtin_amdgcn_readfirstlane(slot);
        first = __builtin_amdgcn_readfirstlane(first);
        len = __builtin_amdgcn_readfirstlane(len);
        count = __builtin_amdgcn_readfirstlane(count);
        asm("" : "+s"(slot), "+s"(first), "+s"(len), "+s"(count));  // (none is used before all are here)
    }
    Seen s;
    s.slot = a.slot ? slot : r;
    s.cap = kv.blocks * MZ_KV_BLK;
    s.base = (long)a.len_add + (a.len ? len : 0);
    s.first = a.first ? max(first, 0) : 0;
    s.count = a.count ? min(max(count, 0), a.tokens) : a.tokens;
    if (s.slot < 0 || s.slot >= kv.slots) s.slot = s.cap = 0;
    return s;
}

// Alignment indices of the query heads h0 .. h0 + n - 1, by all threads of the workgroup: of heads with one index the
// first has it. mine: head_slot[threadIdx.x], requested earlier.
template <int THREADS>
__device__ __forceinline__ void align_indices(const MzKv8Attn& a, int h0, int n, int mine, int (&index)[64]) {
    __shared__ int slots[64];
    const int tid = threadIdx.x;
    for (int j = tid; j < h0 + n; j += THREADS) {
        const int s = j == tid ? mine : a.head_slot[j];
        if (j >= h0) slots[j - h0] = index[j - h0] = s < a.align_heads ? s : -1;
    }
    __syncthreads();
    for (int j = tid; j < h0 + n; j += THREADS) {
        const int s = j == tid ? mine : a.head_slot[j];
        for (int k = max(0, j - h0 + 1); k < n; k++)
            if (slots[k] == s) index[k] = -1;
    }
    __syncthreads();
}

struct Launch {
    int qt, tiles, splits;  // queries of a workgroup / 16, such tiles of a (row, cache head), workgroups that share the blocks
    int waves, own;         // waves of a workgroup; whether each has 16 queries of its own (qt is not used then)
    int kept;               // alignment rows: scores that a workgroup keeps in LDS for each query, 0: in their rows
    int group;              // query heads of a cache head
    unsigned by_heads, by_group, by_splits;  // for dividing by the cache's heads, group and splits (see divided)
};
// x / d for x below 2^31 by r = min(2^32 / d, 2^32 - 1): no more than one too small before the correction (a division by a
// number not known beforehand takes about twenty dependent instructions)
__device__ __forceinline__ int divided(int x, int d, unsigned r) {
    const int q = (int)__umulhi((unsigned)x, r);
    return q + ((q + 1) * (long)d <= x);
}
constexpr int STATE = 66;  // floats of a query's partial state: 64 channels, maximum, sum

// NW waves, which take the blocks in turn, or, with OWN, each 16 QT queries of its own and every block (no alignment rows):
// widening a block is then the four waves' common work, which meet once a block (measured with P as one fp16
// number, 8 prompts of 224 tokens over up to 374 positions: 13.4 us, 15.5 when each made its own, over 1500 positions 42 and 56).
template <int FMT, int QT, bool ALIGN, int NW, bool OWN>
__global__ void __launch_bounds__(64 * NW, OWN ? 5 : QT == 1 ? 4 : 2) attn_kernel(MzKv8 kv, MzKv8Attn a, Launch n) {
    static_assert(!(OWN && ALIGN));
    __shared__ float red[OWN ? 1 : NW][16][68], ms[NW][16], ls[NW][16];
    __shared__ float lse2s[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    // x: (row, cache head), padded to a multiple of the XCDs, so that what shares keys and values shares an XCD; y: the tiles,
    // those that see most first; z: the shares of the blocks
    const int pairs = a.rows * kv.heads, pair = min((int)blockIdx.x, pairs - 1);
    const int tile = n.tiles - 1 - (int)blockIdx.y, split = blockIdx.z, grp = n.group;
    const int r = divided(pair, kv.heads, n.by_heads), kh = pair - r * kv.heads;
    const Seen s = seen_of(kv, a, r);
    // the workgroup's queries, and this wave's
    constexpr int SHARE = OWN ? NW : 1;
    const int nq = a.tokens * grp, w0 = tile * 16 * QT * SHARE, wn = min(w0 + 16 * QT * SHARE, nq);
    const int q0 = OWN ? w0 + 16 * QT * wave : w0, qn = min(q0 + 16 * QT, nq);
    auto token_of = [&](int x) { return divided(x, grp, n.by_group); };
    // (one way out, behind the first loads)
    if ((int)blockIdx.x >= pairs || token_of(w0) >= s.count) return;  // none of its tokens is there
    const int lo_end = s.end(a, token_of(q0)), hi = s.end(a, min(token_of(wn - 1), s.count - 1));
    const int b_lo = s.first / MZ_KV_BLK, nb = max((hi + MZ_KV_BLK - 1) / MZ_KV_BLK - b_lo, 0);
    // (splits is at most 256, nb below 2^20)
    const int b0 = b_lo + (OWN || n.splits == 1 ? 0 : divided(nb * split, n.splits, n.by_splits));
    const int b1 = b_lo + (OWN || n.splits == 1 ? nb : divided(nb * (split + 1), n.splits, n.by_splits));

    const long sh = s.slot * kv.heads + kh;
    int zero = 0;
    asm("" : "+v"(zero));
    const int open_word = kv.open[sh + zero];  // (a vector load: the scalar ones would all be waited for together)
    const unsigned char* kc = kv.k + sh * kv.blocks * MZ_KV_TILE;
    const unsigned char* vc = kv.v + sh * kv.blocks * MZ_KV_TILE;
    const float* ksc = kv.k_scale + sh * kv.blocks;
    const float* vsc = kv.v_scale + sh * kv.blocks;

    extern __shared__ float kept[];  // [query][n.kept]
    __shared__ int index[ALIGN ? 64 : 1];
    const int mine = ALIGN && tid < a.heads ? a.head_slot[tid] : -1;
    f16x8 qf[QT][2];
    int end[QT];  // what a lane's queries see ends here (0: they see nothing),
    unsigned span[QT];  // and has these many positions
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
        end[t] = on ? s.end(a, i) : 0;
        span[t] = max(end[t] - s.first, 0);
        if (span[t] == 0) end[t] = 0;  // (also where the first position is in the block that the end is in)
        al[t] = nullptr;
    }

    // A coded block as it lies. Blocks past this workgroup's share read as zeros, without a memory access: the loads need no
    // branches, around which the compiler would wait for all that is on its way.
    struct Raw {
        u32x4 k[2], v[2];
    };
    const unsigned ktok = 8 * (c >> 2) + (c & 3);  // row c of key tile 0; tile 1 is 4 positions on
    const __amdgpu_buffer_rsrc_t rk = rsrc(kc + (long)b0 * MZ_KV_TILE, (b1 - b0) * MZ_KV_TILE);
    const __amdgpu_buffer_rsrc_t rv = rsrc(vc + (long)b0 * MZ_KV_TILE, (b1 - b0) * MZ_KV_TILE);
    const unsigned kat = ktok * 64 + 16 * g, vat = (c * 4 + g) * 16;
    constexpr int POLICY = QT == 1 && !OWN ? 2 : 0;  // nontemporal where no other workgroup reads the same
    auto fetch = [&](int b, Raw& w) {
        const unsigned o = (unsigned)(b - b0) * MZ_KV_TILE;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            w.k[j] = __builtin_amdgcn_raw_buffer_load_b128(rk, kat + o + 256 * j, 0, POLICY);
            w.v[j] = __builtin_amdgcn_raw_buffer_load_b128(rv, vat + o + 1024 * j, 0, POLICY);
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
    float inf = INFINITY;
    asm("" : "+s"(inf));
    // A block's scales: cs the keys' in the exponent (of two); of the values' the logarithm lg, which goes into P, and the
    // reciprocal rc, which takes it out of the sum again; where it is 0 or no number lg is 0, rc 1, and P's factor is by.
    struct Scales {
        float cs, lg, rc, by;
    };
    // (low: what vf lacks of the open block's fp16 numbers)
    auto products = [&](int b, const f16x8 (&kf)[2][2], const bf16x8 (&vf)[4], const bf16x8 (&low)[4], const Scales& sc, auto open_block) {
        // the open block's fp16 numbers as they were given: any numbers
        constexpr bool given = decltype(open_block)::value;
        const int p0 = b * MZ_KV_BLK + 8 * g;  // this lane's positions
        const bool whole = b * MZ_KV_BLK >= s.first && (b + 1) * MZ_KV_BLK <= lo_end;  // seen by every query
#pragma unroll
        for (int t = 0; t < QT; t++) {
            f32x4 d[2];
#pragma unroll
            for (int j = 0; j < 2; j++) d[j] = mfma16(kf[j][1], qf[t][1], mfma16(kf[j][0], qf[t][0], f32x4{}));
            if (!whole)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if ((unsigned)(p0 - s.first + e) >= span[t]) d[e >> 2][e & 3] = -INFINITY;
            // A block that a query does not see leaves it alone: codes are numbers, but the scales may be none, and so may be
            // what was given.
            const bool any = whole || b * MZ_KV_BLK < end[t];
            const float cs = any ? sc.cs : 1.f;
            if (ALIGN && al[t] != nullptr) {
                const f32x4 x[2] = {d[0] * cs, d[1] * cs};
                if (n.kept) {
                    f32x4* o = (f32x4*)(kept + (16 * t + c) * n.kept + p0 - b0 * MZ_KV_BLK);
                    o[0] = x[0];
                    o[1] = x[1];
                } else {
                    for (int e = 0; e < 8; e++)
                        if (p0 + e >= s.first && p0 + e < min(end[t], a.align_cols)) {
                            if (n.splits > 1) shared_store(al[t] + p0 + e, x[e >> 2][e & 3]);
                            else al[t][p0 + e] = x[e >> 2][e & 3];
                        }
                }
            }
            const float top = cs * fmaxf(fmaxf(larger(d[0][0], d[0][1], inf), larger(d[0][2], d[0][3], inf)),
                                         fmaxf(larger(d[1][0], d[1][1], inf), larger(d[1][2], d[1][3], inf)));
            if (__ballot(top > m[t] + 8.f)) {
                const float mn = fmaxf(m[t], column_max(top)), f = __builtin_amdgcn_exp2f(m[t] - mn);
                m[t] = mn;
                l[t] *= f;
#pragma unroll
                for (int u = 0; u < 4; u++) acc[t][u] *= f;
            }
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __builtin_amdgcn_exp2f(fmaf(d[e >> 2][e & 3], cs, sc.lg - m[t]));
            l[t] += (((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]))) * sc.rc;
            asm volatile("" : "+v"(l[t]));  // (the sum is taken here: later it would need copies of x)
            if (!given && sc.by != 1.f) {
                const float by = any ? sc.by : 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] *= by;
            }
            u32x4 high, rest;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                unsigned h = __builtin_bit_cast(unsigned, bf16x2{(__bf16)x[2 * e], (__bf16)x[2 * e + 1]});
                asm("" : "+v"(h));  // (rounded once)
                const float r0 = x[2 * e] - __builtin_bit_cast(float, h << 16), r1 = x[2 * e + 1] - __builtin_bit_cast(float, h & 0xffff0000u);
                high[e] = h;
                rest[e] = __builtin_bit_cast(unsigned, bf16x2{(__bf16)r0, (__bf16)r1});
            }
            const bf16x8 p = __builtin_bit_cast(bf16x8, high), q = __builtin_bit_cast(bf16x8, rest);
#pragma unroll
            for (int u = 0; u < 4; u++)
                if constexpr (given) {  // by itself: nothing of it where nothing is seen
                    const f32x4 y = weighted(vf[u], p, q, weighted(low[u], p, q, f32x4{}));
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[t][u][e] = any ? acc[t][u][e] + y[e] : acc[t][u][e];
                } else
                    acc[t][u] = weighted(vf[u], p, q, acc[t][u]);
        }
    };
    auto coded = [&](int b, const Raw& w, const Scales& sc) {
        f16x8 kf[2][2];
        bf16x8 vf[4];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            kf[j][0] = widen<FMT>(w.k[j][0], w.k[j][1]);
            kf[j][1] = widen<FMT>(w.k[j][2], w.k[j][3]);
            vf[2 * j] = widen_bf16<FMT>(w.v[j][0], w.v[j][1]);
            vf[2 * j + 1] = widen_bf16<FMT>(w.v[j][2], w.v[j][3]);
        }
        products(b, kf, vf, vf, sc, std::false_type{});
    };
    // Blocks b0 + wave, + NW, ..., or every block: DEPTH or AHEAD of them on their way. The open block, where it is this
    // wave's, comes first; its codes are stale.
    // The scales of 60 of them lie in the lanes of two registers: scalar loads, which come back in any order, would have
    // every block wait for the newest of them.
    constexpr int DEPTH = 2, WINDOW = 60, STEP = OWN ? 1 : NW, AHEAD = 2;
    Raw w[DEPTH];
    const int head = b0 + (OWN ? 0 : wave);
    if constexpr (!OWN)
#pragma unroll
        for (int i = 0; i < DEPTH; i++) fetch(head + STEP * i, w[i]);
    if constexpr (ALIGN) {  // (while they are on their way)
        align_indices<64 * NW>(a, kh * grp, grp, mine, index);
#pragma unroll
        for (int t = 0; t < QT; t++) al[t] = align_row(t);
    }
    if (head < b1) {
        const int tail = head + (b1 - 1 - head) / STEP * STEP;
        Scales lanes;
        auto scales = [&](int b) {
            const int at = min(b + STEP * lane, tail);
            const float ks = ksc[at], vs = vsc[at], cs = scale2 * ks;
            lanes.cs = cs == 0.f ? 1e-37f : cs;  // (all keys 0; what is not seen is -inf times it)
            const float lg = __builtin_amdgcn_logf(vs);
            const bool into = fabsf(lg) < 100.f;
            lanes.lg = into ? lg : 0.f;
            lanes.rc = into ? __builtin_amdgcn_rcpf(vs) : 1.f;
            lanes.by = into ? 1.f : vs;
        };
        auto scales_of = [&](int i) {
            return Scales{lane_value(lanes.cs, i), lane_value(lanes.lg, i), lane_value(lanes.rc, i), lane_value(lanes.by, i)};
        };
        u32x4 raw[AHEAD];
        const auto part = wave < 2 ? rk : rv;
        const unsigned at0 = wave < 2 ? kat + 256 * wave : vat + 1024 * (wave - 2);
        auto take = [&](int i) { return __builtin_amdgcn_raw_buffer_load_b128(part, at0, min(i, tail - b0) * MZ_KV_TILE, 0); };
        if constexpr (OWN)
#pragma unroll
            for (int i = 0; i < AHEAD; i++) raw[i] = take(i);
        scales(head);
        const int open = s.cap ? __builtin_amdgcn_readfirstlane(open_word) - 1 : -1;
        // what this wave's queries see ends here
        const int own_end = !OWN ? hi : q0 < nq && token_of(q0) < s.count ? s.end(a, min(token_of(qn - 1), s.count - 1)) : 0;
        if (open >= b0 && open < b1 && (open - head) % STEP == 0 && open * MZ_KV_BLK < own_end) {
            f16x8 kf[2][2];
            bf16x8 vf[4], low[4];
            const f16* ko = kv.k_open + sh * MZ_KV_TILE;
            const f16* vo = kv.v_open + sh * MZ_KV_TILE;
            u32x4 there;  // what no query of the tile sees may be no number
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int p = open * MZ_KV_BLK + 8 * g + 2 * e;
                there[e] = (p < s.first || p >= hi ? 0u : 0xffffu) | (p + 1 < s.first || p + 1 >= hi ? 0u : 0xffff0000u);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                kf[j >> 1][j & 1] = ld8(ko + (ktok + 4 * (j >> 1)) * 64 + 16 * g + 8 * (j & 1));
                // eleven bits as eight and the other three, both exact
                const u32x4 v = __builtin_bit_cast(u32x4, ld8(vo + ((16 * (j >> 1) + c) * 4 + g) * 16 + 8 * (j & 1)));
                u32x4 v8, v3;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const unsigned y = v[e] & there[e], y8 = y & 0xfff8fff8u;
                    v8[e] = as_bf16(__builtin_bit_cast(f16x2, y8));
                    v3[e] = as_bf16(__builtin_bit_cast(f16x2, y) - __builtin_bit_cast(f16x2, y8));
                }
                vf[j] = __builtin_bit_cast(bf16x8, v8);
                low[j] = __builtin_bit_cast(bf16x8, v3);
            }
            products(open, kf, vf, low, Scales{scale2, 0.f, 1.f, 1.f}, std::true_type{});
        }
        if constexpr (OWN) {
            // Each wave widens a quarter of a block (waves 0 and 1 of the keys) and puts it where all find it, a block
            // ahead; what is behind the last block is that one again.
            __shared__ u32x4 pieces[2][8][64];
            auto put = [&](int b, const u32x4& x) {
                u32x4* o = &pieces[b & 1][2 * wave][lane];
                if (wave < 2) {
                    o[0] = __builtin_bit_cast(u32x4, widen<FMT>(x[0], x[1]));
                    o[64] = __builtin_bit_cast(u32x4, widen<FMT>(x[2], x[3]));
                } else {
                    o[0] = __builtin_bit_cast(u32x4, widen_bf16<FMT>(x[0], x[1]));
                    o[64] = __builtin_bit_cast(u32x4, widen_bf16<FMT>(x[2], x[3]));
                }
            };
            put(0, raw[0]);
            __syncthreads();
            for (int w0 = 0; w0 <= tail - b0; w0 += WINDOW) {
                if (w0) scales(b0 + w0);
                const int w1 = min(w0 + WINDOW, tail - b0 + 1);
                for (int i0 = w0; i0 < w1; i0 += AHEAD)
#pragma unroll
                    for (int j = 0; j < AHEAD; j++) {
                        const int i = i0 + j, b = b0 + i;
                        if (i >= w1) break;
                        raw[j] = take(i + AHEAD);
                        put(i + 1, raw[(j + 1) % AHEAD]);
                        if (b * MZ_KV_BLK < own_end && b != open) {
                            f16x8 kf[2][2];
                            bf16x8 vf[4];
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                kf[k >> 1][k & 1] = __builtin_bit_cast(f16x8, pieces[i & 1][k][lane]);
                                vf[k] = __builtin_bit_cast(bf16x8, pieces[i & 1][4 + k][lane]);
                            }
                            products(b, kf, vf, vf, scales_of(i - w0), std::false_type{});
                        }
                        __syncthreads();
                    }
            }
        } else
            for (int b = head, at = 0; b <= tail; b += STEP * DEPTH, at += DEPTH) {
                if (at == WINDOW) {
                    scales(b);
                    at = 0;
                }
#pragma unroll
                for (int i = 0; i < DEPTH; i++) {
                    const int bi = b + STEP * i;
                    if (bi <= tail && bi != open) coded(bi, w[i], scales_of(at + i));
                    fetch(bi + STEP * DEPTH, w[i]);
                }
            }
    }

    // accumulator u of lane (c, g) holds channels 32 (u / 2) + 8 g + 2 e + u % 2 of query c
    if constexpr (OWN) {
#pragma unroll
        for (int t = 0; t < QT; t++) {
            const int x = q0 + 16 * t + c, i = token_of(x), h = kh * grp + x - i * grp;
            const float ll = column_sum(l[t]), f = ll == 0.f ? 0.f : 1.f / ll;
            if (x >= nq || i >= s.count) continue;
            f16* o = a.out + r * a.out_row + i * a.out_token + h * a.out_head + 8 * g;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const f32x4 y = acc[t][2 * u] * f, z = acc[t][2 * u + 1] * f;
                *(f16x8*)(o + 32 * u) = f16x8{(f16)y[0], (f16)z[0], (f16)y[1], (f16)z[1], (f16)y[2], (f16)z[2], (f16)y[3], (f16)z[3]};
            }
            if (a.lse && g == 0)
                a.lse[((long)r * a.tokens + i) * a.heads + h] = ll == 0.f ? -INFINITY : (m[t] + __builtin_amdgcn_logf(ll)) * LN2;
        }
        return;
    }
    // the waves' states joined, 16 queries at a time, by the first 256 threads
    const int col = tid >> 4 & 15, d4 = (tid & 15) * 4;
    const bool mine256 = NW == 4 || tid < 256;
    // Alignment rows of 16 queries: their scores (in powers of two, get(query, row, position)) to probabilities, 0 where nothing
    // is seen, by all threads, eight of a row's scores a thread at a time and the first ones of four rows.
    constexpr int STRIDE = 64 * NW;
    auto rows = [&](int t) { return (unsigned)__ballot(al[t] != nullptr) & 0xffff; };
    auto row_of_query = [&](int t, int k) {
        const unsigned long at = (unsigned long)al[t];
        return (float*)((unsigned long)(unsigned)__builtin_amdgcn_readlane((int)(at >> 32), k) << 32 |
                        (unsigned)__builtin_amdgcn_readlane((int)at, k));
    };
    auto scores = [&](int t, int k, int p0, float (&x)[8], auto get) {
        const float* row = row_of_query(t, k);
        const int to = min(s.end(a, token_of(q0 + 16 * t + k)), a.align_cols);
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
    auto in_lds = [&](int q, const float*, int p) { return kept[q * n.kept + p - b0 * MZ_KV_BLK]; };
    auto in_place = [&](int, const float* row, int p) { return row[p]; };
    auto in_memory = [&](int, const float* row, int p) { return shared_load(row + p); };
    auto emit = [&](int t, float mm, float ll, f32x4 o, Few& scores, auto get) {
        const int x = q0 + 16 * t + col, i = token_of(x), h = kh * grp + x - i * grp;
        const float inv = ll == 0.f ? 0.f : 1.f / ll, lse2 = ll == 0.f ? -INFINITY : mm + __builtin_amdgcn_logf(ll);
        if (mine256 && x < nq && i < s.count) {
            st4(a.out + r * a.out_row + i * a.out_token + h * a.out_head + d4, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            if (a.lse && d4 == 0) a.lse[((long)r * a.tokens + i) * a.heads + h] = lse2 * LN2;
        }
        if (ALIGN) {
            if (mine256 && d4 == 0) lse2s[col] = lse2;
            __syncthreads();
            probabilities(t, scores, get);
            __syncthreads();
        }
    };
    float* const states = a.work + JOIN_COUNTERS + ((long)pair * n.tiles + tile) * n.splits * (16 * QT) * STATE;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const float lt = column_sum(l[t]);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float* o = &red[wave][c][32 * u + 8 * g];
            const f32x4 x = acc[t][2 * u], y = acc[t][2 * u + 1];
            *(f32x4*)o = f32x4{x[0], y[0], x[1], y[1]};
            *(f32x4*)(o + 4) = f32x4{x[2], y[2], x[3], y[3]};
        }
        if (g == 0) {
            ms[wave][c] = m[t];
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
        if (n.splits == 1) {
            Few x;
            if (n.kept) {
                few_scores(t, ALIGN ? rows(t) : 0, x, in_lds);
                emit(t, mm, ll, o, x, in_lds);
            } else {
                few_scores(t, ALIGN ? rows(t) : 0, x, in_place);
                emit(t, mm, ll, o, x, in_place);
            }
        }
        else if (mine256 && q0 + 16 * t + col < nq) {
            float* w = states + (split * (16 * QT) + 16 * t + col) * STATE;
            shared_store(w + d4, o[0], o[1]);
            shared_store(w + d4 + 2, o[2], o[3]);
            if (d4 == 0) shared_store(w + 64, mm, ll);
        }
        if (ALIGN && n.splits > 1 && n.kept)  // the share's scores to where the last workgroup finds them
            for (unsigned has = rows(t); has; has &= has - 1) {
                const int k = __ffs(has) - 1;
                float* const row = row_of_query(t, k);
                for (int p = b0 * MZ_KV_BLK + tid; p < min(b1 * MZ_KV_BLK, a.align_cols); p += STRIDE)
                    shared_store(row + p, in_lds(16 * t + k, row, p));
            }
        if (t + 1 < QT) __syncthreads();
    }
    if (n.splits == 1 || !last_of((unsigned*)a.work + (long)pair * n.tiles + tile, n.splits)) return;
    // the last of the workgroups that share these queries joins their states
#pragma unroll
    for (int t = 0; t < QT; t++) {
        float mm = NOTHING, ll = 0.f;
        f32x4 o = {};
        Few x;
        few_scores(t, ALIGN ? rows(t) : 0, x, in_memory);  // (they come with the states)
        if (mine256 && q0 + 16 * t + col < nq)
            for (int k0 = 0; k0 < n.splits; k0 += 4) {
                float2 y[4][3];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float* w = states + (min(k0 + k, n.splits - 1) * (16 * QT) + 16 * t + col) * STATE;
                    y[k][0] = shared_load2(w + d4);
                    y[k][1] = shared_load2(w + d4 + 2);
                    y[k][2] = shared_load2(w + 64);
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (k0 + k >= n.splits) continue;
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

// LDS for the scores of alignment rows: 1504 positions of five queries fit, so that three workgroups share a CU, or of sixteen
// where each has one to itself
constexpr long KEPT_FLOATS = 8192, KEPT_FLOATS_ALONE = 24576;
long kept_queries(const Launch& n, long nq) { return std::min(nq, 16L * n.qt); }

// Measured, us, 20 heads unless stated, no alignment rows; a unit is a tile of a (row, cache head).
// Up to 16 queries: a tile of 16, and no more units than CUs: eight waves each instead of four (1500 positions, 160 units
// 10.1 / 11.0, five beams of 256 units 10.9 / 11.3, but 260 units 15.8 / 14.5, 640 units 24.8 / 23.5), and with fewer than
// half as many, the blocks shared by more workgroups until there is one a CU or a wave has about a block left (1500 positions
// of one row 9.5 with one workgroup, 8.8 with 2, 7.6 with 4; 80 units 9.7, 8.8 with 3, 10.0 with 4; 16,000 positions of 48
// units 47 with one, 20.0 with 5, 22.6 with 8).
// More queries: each wave 16 of its own, or tiles of 32 whose waves take the blocks in turn. Under a causal mask the first where
// that gives every CU a workgroup (224-token prompts of 8 rows 13.3 / 14.6, 40 tokens of 16 rows 8.7 / 10.2; but of one row
// 10.2 / 7.6, of 3 rows 10.4 / 8.9). Without one all workgroups take the same time, and the first needs three and a half a CU,
// or a last round of them leaves most CUs idle (224 tokens over 1500 positions: 7 rows, 2.2 workgroups a CU, 45.8 / 34.4, 8 rows
// 46.0 / 39.6, 10 rows, 3.1, 56 / 47, 16 rows, 5.0, 68 / 74, 32 rows 136 / 150; over 374 positions 10 rows 21.2 / 20.9, 24 rows of
// 128 tokens, 3.8, 22.1 / 26.4; the other way 32 rows of 40 tokens, 2.5, 17.2 / 19.4).
Launch attn_shape(const MzKv8& kv, const MzKv8Attn& a) {
    const long nq = (long)a.tokens * (a.heads / kv.heads), cus = mz_cu_count(), pairs = (long)a.rows * kv.heads;
    auto inverse = [](int d) { return (unsigned)std::min((1ULL << 32) / d, 0xffffffffULL); };
    Launch n{};
    n.group = a.heads / kv.heads;
    n.by_heads = inverse(kv.heads);
    n.by_group = inverse(n.group);
    n.waves = 4;
    n.splits = 1;
    n.own = !a.align && nq > 16 && 2 * pairs * ((nq + 63) / 64) >= (a.causal ? 2 : 7) * cus;
    if (n.own) {
        n.tiles = (int)((nq + 63) / 64);
        return n;
    }
    n.qt = nq <= 16 ? 1 : 2;
    n.tiles = (int)((nq + 16 * n.qt - 1) / (16 * n.qt));
    const long units = pairs * n.tiles;
    if (units <= cus && n.qt == 1) n.waves = 8;
    n.splits = (int)std::max(1L, std::min({cus / units, (long)kv.blocks / 10, 256L}));
    n.by_splits = inverse(n.splits);
    const long keep = ((long)kv.blocks + n.splits - 1) / n.splits * MZ_KV_BLK;
    n.kept = a.align && keep * kept_queries(n, nq) <= (units * n.splits <= cus ? KEPT_FLOATS_ALONE : KEPT_FLOATS) ? (int)keep : 0;
    return n;
}
static_assert(JOIN_COUNTERS >= 1024, "units that are shared have a counter each: fewer than the CUs");

template <int FMT, bool ALIGN>
void attn_launch(hipStream_t s, const MzKv8& kv, const MzKv8Attn& a, const Launch& n) {
    const size_t lds = (size_t)n.kept * kept_queries(n, (long)a.tokens * n.group) * 4;
    const dim3 grid(((long)a.rows * kv.heads + 7) / 8 * 8, n.tiles, n.splits);
    if constexpr (!ALIGN)
        if (n.own) {
            hipLaunchKernelGGL((attn_kernel<FMT, 1, false, 4, true>), grid, dim3(256), 0, s, kv, a, n);
            return;
        }
    if (n.qt == 2) hipLaunchKernelGGL((attn_kernel<FMT, 2, ALIGN, 4, false>), grid, dim3(256), lds, s, kv, a, n);
    else if (n.waves == 4) hipLaunchKernelGGL((attn_kernel<FMT, 1, ALIGN, 4, false>), grid, dim3(256), lds, s, kv, a, n);
    else hipLaunchKernelGGL((attn_kernel<FMT, 1, ALIGN, 8, false>), grid, dim3(512), lds, s, kv, a, n);
}

}  // namespace

// (a launch has fewer than 2^32 threads along x, and 2^16 workgroups along y and z)
bool mz_kv8_io_fits(const MzKv8& kv, const MzKv8Io& a) { return a.rows <= 65535 && kv.heads <= 65535; }

bool mz_kv8_attn_fits(const MzKv8& kv, const MzKv8Attn& a) {
    const long nq = (long)a.tokens * (a.heads / kv.heads);
    return (long)a.rows * kv.heads < (1L << 23) - 8 && nq <= 16L * 65535;
}

size_t mz_kv8_attn_work(const MzKv8& kv, const MzKv8Attn& a) {
    const Launch n = attn_shape(kv, a);
    return n.splits > 1 ? ((size_t)a.rows * kv.heads * n.tiles * n.splits * 16 * n.qt * STATE + JOIN_COUNTERS) * 4 : 0;
}

hipError_t mz_kv8_write_launch(hipStream_t s, const MzKv8& kv, const MzKv8Io& a) {
    const int per = write_per(kv, a);
    const dim3 grid(write_groups(kv, a, per), kv.heads, a.rows), block(a.tokens == 1 ? 128 : 256);  // (one token: one block)
    if (kv.format == I8) hipLaunchKernelGGL(write_kernel<I8>, grid, block, 0, s, kv, a, per);
    else hipLaunchKernelGGL(write_kernel<E4M3>, grid, block, 0, s, kv, a, per);
    return hipGetLastError();
}

hipError_t mz_kv8_read_launch(hipStream_t s, const MzKv8& kv, const MzKv8Io& a) {
    const dim3 grid((spanned(kv, a) + 1) / 2, kv.heads, a.rows);
    if (kv.format == I8) hipLaunchKernelGGL(read_kernel<I8>, grid, dim3(256), 0, s, kv, a);
    else hipLaunchKernelGGL(read_kernel<E4M3>, grid, dim3(256), 0, s, kv, a);
    return hipGetLastError();
}

hipError_t mz_kv8_attn_launch(hipStream_t s, const MzKv8& kv, const MzKv8Attn& a) {
    const Launch n = attn_shape(kv, a);
    if (kv.format == I8) a.align ? attn_launch<I8, true>(s, kv, a, n) : attn_launch<I8, false>(s, kv, a, n);
    else a.align ? attn_launch<E4M3, true>(s, kv, a, n) : attn_launch<E4M3, false>(s, kv, a, n);
    return hipGetLastError();
}
