// Key/value caches held in 8 bits: writing, reading back, and attention over them (layout and definitions: mz_kv8 in
// mimizuku.h). Plain kernels: one wave per (row, head), or per query.
#include "mz_common.h"
#include "mz_kernels.h"

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

template <int FMT>
__global__ void __launch_bounds__(64) attn_kernel(MzKv8 kv, MzKv8Attn a) {
    __shared__ float qs[64], ps[64];
    const int lane = threadIdx.x;
    long id = blockIdx.x;
    const int h = id % a.heads, i = id / a.heads % a.tokens, r = id / a.heads / a.tokens;
    if (a.count && i >= a.count[r]) return;
    const long slot = a.slot ? a.slot[r] : r, cap = (long)kv.blocks * MZ_KV_BLK;
    const bool there = slot >= 0 && slot < kv.slots;
    long end = (long)a.len_add + (a.len ? a.len[(long)r * a.len_stride] : 0) + (a.causal ? i : 0);
    end = there ? min(max(end, 0L), cap) : 0;
    const int lo = a.first ? max(a.first[r], 0) : 0, hi = (int)end;
    const long sh = (there ? slot : 0) * kv.heads + h / (a.heads / kv.heads);
    const int open = kv.open[sh];
    int as = a.head_slot ? a.head_slot[h] : -1;
    if (as >= a.align_heads) as = -1;
    for (int j = 0; j < h && as >= 0; j++)
        if (a.head_slot[j] == as) as = -1;
    float* al = as >= 0 ? a.align + ((((long)r * a.tokens + i) * a.align_heads + as) * a.align_cols) : nullptr;
    qs[lane] = (float)a.q[r * a.q_row + i * a.q_token + h * a.q_head + lane];
    __syncthreads();
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int p0 = lo; p0 < hi; p0 += 64) {
        const int n = min(64, hi - p0);
        float s = -INFINITY;
        if (lane < n) {
            const int p = p0 + lane, b = p / MZ_KV_BLK, t = p % MZ_KV_BLK;
            const long e = (sh * kv.blocks + b) * MZ_KV_TILE + t * 64;
            s = 0.f;
            for (int d = 0; d < 64; d++)
                s = fmaf(qs[d], open == b + 1 ? (float)kv.k_open[sh * MZ_KV_TILE + t * 64 + d] : code_value<FMT>(kv.k[e + d]), s);
            s *= a.scale * (open == b + 1 ? 1.f : kv.k_scale[sh * kv.blocks + b]);
            if (al && p < a.align_cols) al[p] = s;
        }
        const float mn = fmaxf(m, wave_max(s));
        const float e = lane < n ? expf(s - mn) : 0.f, f = m == mn ? 1.f : expf(m - mn);
        ps[lane] = e;
        __syncthreads();
        l = l * f + wave_sum(e);
        o *= f;
        for (int j = 0; j < n; j++) {
            const int p = p0 + j, b = p / MZ_KV_BLK, t = p % MZ_KV_BLK;
            const float v = open == b + 1 ? (float)kv.v_open[sh * MZ_KV_TILE + v_at(t, lane)]
                                          : code_value<FMT>(kv.v[(sh * kv.blocks + b) * MZ_KV_TILE + v_at(t, lane)]) * kv.v_scale[sh * kv.blocks + b];
            o = fmaf(ps[j], v, o);
        }
        __syncthreads();
        m = mn;
    }
    a.out[r * a.out_row + i * a.out_token + h * a.out_head + lane] = (f16)(hi > lo ? o / l : 0.f);
    const float lse = m + logf(l);
    if (a.lse && lane == 0) a.lse[((long)r * a.tokens + i) * a.heads + h] = hi > lo ? lse : -INFINITY;
    if (al)
        for (int p = lane; p < a.align_cols; p += 64) al[p] = p >= lo && p < hi ? expf(al[p] - lse) : 0.f;
}

}  // namespace

long mz_kv8_write_grid(const MzKv8& kv, const MzKv8Io& a) { return (long)a.rows * kv.heads; }
long mz_kv8_read_grid(const MzKv8& kv, const MzKv8Io& a) { return (long)a.rows * kv.heads; }
long mz_kv8_attn_grid(const MzKv8& kv, const MzKv8Attn& a) { return (long)a.rows * a.tokens * a.heads; }
size_t mz_kv8_attn_work(const MzKv8&, const MzKv8Attn&) { return 0; }

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
    const dim3 grid(mz_kv8_attn_grid(kv, a));
    if (kv.format == I8) hipLaunchKernelGGL(attn_kernel<I8>, grid, dim3(64), 0, s, kv, a);
    else hipLaunchKernelGGL(attn_kernel<E4M3>, grid, dim3(64), 0, s, kv, a);
    return hipGetLastError();
}
