// Products with 4-bit weights (mz_w4 in mimizuku.h): y[m, n] = sum over the groups g of a row of weights of
//     scale[n, g] * (sum over the columns k of g of code[n, k] x[m, k]).
// A code is a whole number of -8 .. 7, exact in fp16, so the sums of a group run on the matrix cores (products of two fp16
// numbers are exact in fp32, and so is the accumulator's format), and a group's scale, fp16 too, is applied to its sum in fp32: no
// weight is ever rounded, and nothing rounds to fewer bits than 32 before the result is stored.
// Few rows of x are bound by the bytes of the weights, 4 bits and 16 / group each, and below that by the launch; from about 32
// rows on, by turning codes into fp16 (9 operations for 8 codes) and by reading x from LDS; hundreds of rows of x by the
// rate at which both feed the matrix cores.
//
// Times here are of a call among 40 back to back, fp16 results (logits fp32), the weights each time others of up to 16 that are
// alike, so that caches hold the small ones only. Both sides of a rule are of one run. A profiler runs launches apart: 1792 x
// 5120 x 1280 with GELU takes 39 to 40 us there, 35 among others.
#include <algorithm>

#include "mz_common.h"
#include "mz_kernels.h"

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Where column 32 s + 8 j + e of the 128 columns of an entry is: word s of entry 16 j + row, bits 4 (e / 2) + 16 (e % 2).
__device__ __forceinline__ int bit_of(int e) { return 4 * (e >> 1) + 16 * (e & 1); }

// A wave: 16 rows x 128 columns; lane 16 j + i has row i, columns 32 s + 8 j .. + 7 (s < 4), which are what its 16 bytes of
// codes hold. A group of 32 columns is a word of four lanes (i + 16 j), one of 64 two words, one of 128 all four.
__global__ void __launch_bounds__(256) pack_kernel(MzW4 w, const f16* src, long ld) {
    const int lane = threadIdx.x & 63, i = lane & 15, j = lane >> 4, chunks = w.k / 128;
    const long entry = (long)blockIdx.x * 4 + (threadIdx.x >> 6), tiles = (w.n + 15) / 16;
    if (entry >= tiles * chunks) return;
    const long t = entry / chunks;
    const int c = (int)(entry - t * chunks);
    const bool there = t * 16 + i < w.n;
    const f16* p = src + (there ? t * 16 + i : 0) * ld + c * 128 + 8 * j;
    f16x8 x[4];
    float hi[4], lo[4];
    bool bad[4];
#pragma unroll
    for (int s = 0; s < 4; s++) {
        x[s] = there ? ld8(p + 32 * s) : f16x8{};
        hi[s] = lo[s] = (float)x[s][0];
        bad[s] = false;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = (float)x[s][e];
            hi[s] = fmaxf(hi[s], v);
            lo[s] = fminf(lo[s], v);
            bad[s] |= !(fabsf(v) <= 65504.f);
        }
#pragma unroll
        for (int o = 16; o < 64; o *= 2) {
            hi[s] = fmaxf(hi[s], __shfl_xor(hi[s], o));
            lo[s] = fminf(lo[s], __shfl_xor(lo[s], o));
            bad[s] |= __shfl_xor((int)bad[s], o) != 0;
        }
    }
    const int words = w.group / 32;  // of a group
    u32x4 q;
    f16 scale[4];
#pragma unroll
    for (int s = 0; s < 4; s++) {
        float h = hi[s], l = lo[s];
        bool b = bad[s];
#pragma unroll
        for (int z = 0; z < 4; z++)
            if (z / words == s / words) {
                h = fmaxf(h, hi[z]);
                l = fminf(l, lo[z]);
                b |= bad[z];
            }
        scale[s] = b ? (f16)NAN : (f16)((h > -l ? h : l) * -0.125f);
        const float d = (float)scale[s];
        unsigned word = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // (a quotient of two fp16 numbers is exactly halfway between whole numbers, and then exact, or 2^-13 away)
            const float y = b || d == 0.f ? 0.f : rintf((float)x[s][e] / d);
            word |= (unsigned)((int)fminf(fmaxf(y, -8.f), 7.f) + 8) << bit_of(e);
        }
        q[s] = word;
    }
    *(u32x4*)(w.codes + (entry * 64 + lane) * 16) = q;
    const int groups = 128 / w.group;
    if (j == 0)
#pragma unroll
        for (int s = 0; s < 4; s++)
            if (s % words == 0) w.scales[(entry * 16 + i) * groups + s / words] = scale[s];
}

__global__ void __launch_bounds__(256) unpack_kernel(MzW4 w, f16* dst, long ld) {
    const int lane = threadIdx.x & 63, i = lane & 15, j = lane >> 4, chunks = w.k / 128;
    const long entry = (long)blockIdx.x * 4 + (threadIdx.x >> 6), tiles = (w.n + 15) / 16;
    if (entry >= tiles * chunks) return;
    const long t = entry / chunks;
    const int c = (int)(entry - t * chunks);
    if (t * 16 + i >= w.n) return;
    const u32x4 q = *(const u32x4*)(w.codes + (entry * 64 + lane) * 16);
    const int words = w.group / 32, groups = 128 / w.group;
#pragma unroll
    for (int s = 0; s < 4; s++) {
        const float d = (float)w.scales[(entry * 16 + i) * groups + s / words];
        f16x8 y;
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = (f16)((float)((int)(q[s] >> bit_of(e) & 15) - 8) * d);
        *(f16x8*)(dst + (t * 16 + i) * ld + c * 128 + 32 * s + 8 * j) = y;
    }
}

// ---------------------------------------------------------------- products

// the eight codes of a word, as they are: 1024 + (c + 8) and 1024 + 16 (c + 8) are fp16 numbers whose low bits are c + 8
struct Codes {
    // (Numbers that the compiler does not know: with those it knows, taking the bits and setting the others are two instructions
    // instead of one. 1 x 51866 x 1280 takes 10.1 us, 11.0 with two. `known` where the registers for the results do not suffice.)
    unsigned one = 0x000F000Fu, sixteen = 0x00F000F0u, magic = 0x64006400u;
    __device__ __forceinline__ explicit Codes(bool known) {
        if (known) return;
        asm("" : "+s"(one), "+s"(sixteen));
        asm("" : "+v"(magic));
    }
    __device__ __forceinline__ f16x8 operator()(unsigned q) const {
        const unsigned q8 = q >> 8;
        const f16x2 off1 = {(f16)-1032.f, (f16)-1032.f}, off16 = {(f16)-72.f, (f16)-72.f}, by = {(f16)0.0625f, (f16)0.0625f};
        const f16x2 a = __builtin_bit_cast(f16x2, (q & one) | magic) + off1;
        const f16x2 b = __builtin_bit_cast(f16x2, (q & sixteen) | magic) * by + off16;
        const f16x2 c = __builtin_bit_cast(f16x2, (q8 & one) | magic) + off1;
        const f16x2 d = __builtin_bit_cast(f16x2, (q8 & sixteen) | magic) * by + off16;
        return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
};

template <int G>  // groups of 128 columns
struct Scales {
    f16 v[G];
};
template <int G>
__device__ __forceinline__ Scales<G> scales_at(const f16* p) {
    if constexpr (G == 4) return __builtin_bit_cast(Scales<4>, *(const f16x4*)p);
    else if constexpr (G == 2) return __builtin_bit_cast(Scales<2>, *(const f16x2*)p);
    else return Scales<1>{*p};
}

__device__ __forceinline__ float bias_of(const MzW4Linear& a, long n) { return a.bias ? (float)a.bias[n] : 0.f; }

// the results of row of weights n for rows m .. m + N - 1 of x, those that there are
template <int N, typename Y>
__device__ __forceinline__ void finish(const MzW4Linear& a, int m, long n, float bias, Y y) {
    const long o = m * a.ldo + n;
    switch (a.epilogue) {
        case 0:
#pragma unroll
            for (int e = 0; e < N; e++)
                if (m + e < a.m) ((f16*)a.out)[o + e * a.ldo] = (f16)(y(e) + bias);
            break;
        case 1:
#pragma unroll
            for (int e = 0; e < N; e++)
                if (m + e < a.m) ((f16*)a.out)[o + e * a.ldo] = (f16)gelu_erf_h(y(e) + bias);
            break;
        case 2: {
            float* out = (float*)a.out + o;
            float old[N];
#pragma unroll
            for (int e = 0; e < N; e++) old[e] = out[m + e < a.m ? e * a.ldo : 0];
#pragma unroll
            for (int e = 0; e < N; e++)
                if (m + e < a.m) out[e * a.ldo] = old[e] + (y(e) + bias);
            break;
        }
        default:
#pragma unroll
            for (int e = 0; e < N; e++)
                if (m + e < a.m) ((float*)a.out)[o + e * a.ldo] = y(e) + bias;
    }
}

// One entry, 16 rows of weights x 128 columns, times 16 MT rows of x: operand lane 16 j + i holds row i, columns 32 s + 8 j .. of
// either; the result's lane 16 j + i holds column i (a row of weights) and rows 4 j .. 4 j + 3 (of x).
template <int MT, int G, typename X>
__device__ __forceinline__ void entry_product(const Codes& numbers, u32x4 q, Scales<G> scale, X x, f32x4 (&sum)[MT]) {
#pragma unroll
    for (int g = 0; g < G; g++) {
        f32x4 part[MT];
#pragma unroll
        for (int z = 0; z < 4 / G; z++) {
            const int s = g * (4 / G) + z;
            const f16x8 w = numbers(q[s]);
#pragma unroll
            for (int t = 0; t < MT; t++) part[t] = mfma16(x(t, s), w, z ? part[t] : f32x4{});
        }
        const float d = (float)scale.v[g];
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum[t][e] = fmaf(part[t][e], d, sum[t][e]);
    }
}

// 16 bytes of each lane straight into LDS, lane after lane from `to` on
__device__ __forceinline__ void to_lds(const f16* from, u32x4* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// Few rows of weights: a workgroup takes 16 of them, its waves the entries in turn, x from memory (which its caches hold); their
// sums meet in LDS. 1 x 5120 x 1280 (rows of x, rows of weights, columns), groups of 64: 4.2 us, of which launch and two
// dependent reads are most; 8 x 1280 x 5120: 5.8 us. Requesting several entries ahead did not help: each wave has two or three.
template <int MT, int G>
__global__ void __launch_bounds__(MT == 4 ? 512 : 1024) split_kernel(MzW4 w, MzW4Linear a) {
    constexpr int LD = 68;  // (of 64 results: four rows of x 4 banks apart, so that reading 16 columns of 4 rows meets no conflict)
    extern __shared__ float red[];  // [wave][4 MT][LD]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x / 64;
    const int i = lane & 15, j = lane >> 4, chunks = w.k / 128, m0 = blockIdx.y * 16 * MT;
    const long t = blockIdx.x;
    const f16* x[MT];
#pragma unroll
    for (int u = 0; u < MT; u++) x[u] = a.x + min(m0 + 16 * u + i, a.m - 1) * a.ldx + 8 * j;
    const Codes numbers(false);
    f32x4 sum[MT] = {};
    for (int c = wave; c < chunks; c += waves) {
        const long entry = t * chunks + c;
        const u32x4 q = *(const u32x4*)(w.codes + (entry * 64 + lane) * 16);
        const Scales<G> scale = scales_at<G>(w.scales + (entry * 16 + i) * G);
        f16x8 v[MT][4];
#pragma unroll
        for (int u = 0; u < MT; u++)
#pragma unroll
            for (int s = 0; s < 4; s++) v[u][s] = ld8(x[u] + c * 128 + 32 * s);
        entry_product<MT, G>(numbers, q, scale, [&](int u, int s) { return v[u][s]; }, sum);
    }
#pragma unroll
    for (int u = 0; u < MT; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) red[(wave * 4 * MT + 4 * u + e) * LD + lane] = sum[u][e];
    __syncthreads();
    for (int o = threadIdx.x; o < 256 * MT; o += blockDim.x) {
        const int n = o & 15, m = o >> 4;  // row m of a tile of x is result 16 (m / 4) + n of m % 4
        const int at = (4 * (m >> 4) + (m & 3)) * LD + 16 * (m >> 2 & 3) + n;
        float y = 0.f;
        for (int k = 0; k < waves; k++) y += red[k * 4 * MT * LD + at];
        if (m0 + m < a.m && t * 16 + n < w.n) finish<1>(a, m0 + m, t * 16 + n, bias_of(a, t * 16 + n), [&](int) { return y; });
    }
}

// Many rows of weights: x lies in LDS, in the order of operands, and each wave takes 16 rows of weights and all of their columns,
// the next entries on their way. 51866 x 1280, groups of 32: 10.1 us for one row (3.7 TB/s, of weights that no cache held), 10.8
// for 8, 11.1 for 16, 15.7 for 32 (2.8 TB/s), 23.7 for 64: no unit bounds these, x goes into LDS whole before the first product, in
// the one workgroup that a CU then has room for, and is read again for every 16 rows of weights. Three, four and five entries ahead
// took 10.9, 11.1 and 11.1 us for the one row when two took 10.8, ten 13.7: more registers, and no wave waits less for its first.
template <int MT, int G>
__global__ void __launch_bounds__(1024) row_kernel(MzW4 w, MzW4Linear a) {
    extern __shared__ u32x4 xs[];  // [chunk][s][MT][64]
    constexpr int AHEAD = 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x / 64;
    const int i = lane & 15, j = lane >> 4, chunks = w.k / 128, m0 = blockIdx.y * 16 * MT, tiles = (w.n + 15) / 16;
    const int t = blockIdx.x * waves + wave, tt = min(t, tiles - 1);
    // entries past the last read as zeros, without a memory access: loads need no branches
    const auto rc = rsrc(w.codes + (long)tt * chunks * 1024, chunks * 1024);
    const auto rs = rsrc(w.scales + (long)tt * chunks * 16 * G, chunks * 16 * G * 2);
    u32x4 q[AHEAD];
    Scales<G> scale[AHEAD];
    auto fetch = [&](int c, int to) {
        q[to] = __builtin_amdgcn_raw_buffer_load_b128(rc, c * 1024 + lane * 16, 0, 2);
        const int at = (c * 16 + i) * G * 2;
        if constexpr (G == 4) scale[to] = __builtin_bit_cast(Scales<4>, __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, 2));
        else if constexpr (G == 2) scale[to] = __builtin_bit_cast(Scales<2>, __builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 2));
        else scale[to] = __builtin_bit_cast(Scales<1>, __builtin_amdgcn_raw_buffer_load_b16(rs, at, 0, 2));
    };
#pragma unroll
    for (int d = 0; d < AHEAD; d++) fetch(d, d);
    for (int f = wave; f < chunks * 4 * MT; f += waves) {
        const int u = f % MT, c4 = f / MT;  // 32 columns
        xs[f * 64 + lane] = __builtin_bit_cast(u32x4, ld8(a.x + min(m0 + 16 * u + i, a.m - 1) * a.ldx + c4 * 32 + 8 * j));
    }
    __syncthreads();
    const Codes numbers(false);
    f32x4 sum[MT] = {};
    for (int c0 = 0; c0 < chunks; c0 += AHEAD)
#pragma unroll
        for (int d = 0; d < AHEAD; d++) {
            const int c = c0 + d;
            if (c < chunks)
                entry_product<MT, G>(numbers, q[d], scale[d], [&](int u, int s) { return __builtin_bit_cast(f16x8, xs[((c * 4 + s) * MT + u) * 64 + lane]); }, sum);
            fetch(c + AHEAD, d);
        }
    const int n = t * 16 + i;
    if (t >= tiles || n >= w.n) return;
    const float bias = bias_of(a, n);
#pragma unroll
    for (int u = 0; u < MT; u++) {
        const int m = m0 + 16 * u + 4 * j;
        if (m < a.m) finish<4>(a, m, n, bias, [&](int e) { return sum[u][e]; });
    }
}

// Many rows of x: a workgroup takes 16 MT WM rows of x times 16 NT WN of weights, WM x WN waves. 128 columns at a time: those of x
// go straight into LDS, in two buffers, the weights' codes into registers. 1792 x 5120 x 1280, groups of 128: 31.6 to 33.6 us
// (700 to 744 TFLOP/s; a library's product of fp16 weights 27.6), of 64: 37.4, of 32: 40.3; 448 rows 13.8, 14.6 and 16.6; 4096 x
// 4096 x 4096, groups of 128: 144 us (953). What bounds it is the vector unit next to the matrix cores: codes turned into numbers
// by every row of waves, scales applied group by group.
template <int MT, int NT, int WM, int WN, int G>
__global__ void __launch_bounds__(64 * WM * WN, 2) tile_kernel(MzW4 w, MzW4Linear a) {
    extern __shared__ u32x4 xs[];  // [2][rows][16 pieces of 8 columns, piece p of row r at p ^ r % 16]
    constexpr int ROWS = 16 * MT * WM, PER = ROWS / (4 * WM * WN);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, j = lane >> 4, chunks = w.k / 128, tiles = (w.n + 15) / 16;
    const int m0 = blockIdx.y * ROWS, wm = wave % WM * 16 * MT, t0 = blockIdx.x * WN * NT + wave / WM * NT;
    // a wave loads four rows at a time, 16 lanes a row
    const f16* from[PER];
#pragma unroll
    for (int z = 0; z < PER; z++) {
        const int r = 4 * (z * WM * WN + wave) + j;
        from[z] = a.x + min(m0 + r, a.m - 1) * a.ldx + 8 * (i ^ (r & 15));
    }
    auto load_x = [&](int c) {
#pragma unroll
        for (int z = 0; z < PER; z++) to_lds(from[z] + c * 128, xs + (c & 1) * ROWS * 16 + 64 * (z * WM * WN + wave));
    };
    u32x4 q[NT];
    Scales<G> scale[NT];
    auto load_w = [&](int c) {
#pragma unroll
        for (int u = 0; u < NT; u++) {
            const long entry = (long)min(t0 + u, tiles - 1) * chunks + c;
            q[u] = *(const u32x4*)(w.codes + (entry * 64 + lane) * 16);
            scale[u] = scales_at<G>(w.scales + (entry * 16 + i) * G);
        }
    };
    // The widest tile has hardly enough registers: groups of 64 keep the numbers that the compiler knows (2000 x 4800 x 2560 69 us,
    // 81 to 83 otherwise, with registers spilled), the others keep it from mixing the steps (1792 x 5120 x 1280, groups of 128, 31.6
    // us, 38.7 mixed; groups of 32 take 40.2 either way).
    constexpr bool APART = G != 2;
    const Codes numbers(NT == 5 && !APART);
    f32x4 sum[MT][NT] = {};
    load_x(0);
    load_w(0);
    for (int c = 0; c < chunks; c++) {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's loads of x have arrived,
        __syncthreads();                     // everyone's have, and nobody reads the other buffer any more
        u32x4 qc[NT];
        Scales<G> sc[NT];
#pragma unroll
        for (int u = 0; u < NT; u++) qc[u] = q[u], sc[u] = scale[u];
        if (c + 1 < chunks) {
            load_x(c + 1);
            load_w(c + 1);
        }
        const u32x4* buf = xs + (c & 1) * ROWS * 16;
        f32x4 part[MT][NT];
#pragma unroll
        for (int s = 0; s < 4; s++) {
            if (APART) __builtin_amdgcn_sched_barrier(0);
            f16x8 x[MT];
#pragma unroll
            for (int u = 0; u < MT; u++) x[u] = __builtin_bit_cast(f16x8, buf[(wm + 16 * u + i) * 16 + ((4 * s + j) ^ i)]);
#pragma unroll
            for (int v = 0; v < NT; v++) {
                const f16x8 y = numbers(qc[v][s]);
#pragma unroll
                for (int u = 0; u < MT; u++) part[u][v] = mfma16(x[u], y, s % (4 / G) ? part[u][v] : f32x4{});
                if (s % (4 / G) == 4 / G - 1) {
                    const float d = (float)sc[v].v[s / (4 / G)];
#pragma unroll
                    for (int u = 0; u < MT; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sum[u][v][e] = fmaf(part[u][v][e], d, sum[u][v][e]);
                }
            }
        }
    }
#pragma unroll
    for (int v = 0; v < NT; v++) {
        const int n = (t0 + v) * 16 + i;
        if (n >= w.n) continue;
        const float bias = bias_of(a, n);
#pragma unroll
        for (int u = 0; u < MT; u++) {
            const int m = m0 + wm + 16 * u + 4 * j;
            if (m < a.m) finish<4>(a, m, n, bias, [&](int e) { return sum[u][v][e]; });
        }
    }
}

int blocks(long x, long per) { return (int)((x + per - 1) / per); }

template <int G>
void linear_launch(hipStream_t s, const MzW4& w, const MzW4Linear& a) {
    const int tiles = blocks(w.n, 16), chunks = w.k / 128, cus = mz_cu_count();
    // Tiles, where there are enough of 64 x 64 for a quarter of the CUs: 224 x 1280 x 5120 (80 of them) takes 24.7 us, 32.0 by
    // split_kernel; 128 x 1280 x 5120 (40) 24.8 and 21.0.
    if (a.m > 64 && (long)blocks(a.m, 64) * blocks(w.n, 64) >= cus / 4) {
        // Of the widths, eight waves a CU, the one whose last round of workgroups leaves the least idle (16 more columns stand for
        // the rows of x; 64: several workgroups a CU, which take 1.15 times as long for a result). 1792 x 5120 x 1280: 33.6 us with
        // 320, 47.5, 37.8, 40.3 and 37.7 with 256, 192, 128 and 64; 448 x 5120 x 1280: 27.6, 23.8, 19.3, 14.7 and 13.9.
        int best = 64;
        double least = 1.15 * blocks(a.m, 64) * blocks(w.n, 64) * 64 * 64 / cus + 64 * 64;
        for (int bn : {320, 256, 192, 128}) {
            const double cost = (double)blocks((long)blocks(a.m, 128) * blocks(w.n, bn), cus) * 128 * (bn + 16);
            if (cost < least) least = cost, best = bn;
        }
        const dim3 grid(blocks(w.n, best), blocks(a.m, best == 64 ? 64 : 128));
        if (best == 320) hipLaunchKernelGGL((tile_kernel<4, 5, 2, 4, G>), grid, dim3(512), 2 * 128 * 256, s, w, a);
        else if (best == 256) hipLaunchKernelGGL((tile_kernel<4, 4, 2, 4, G>), grid, dim3(512), 2 * 128 * 256, s, w, a);
        else if (best == 192) hipLaunchKernelGGL((tile_kernel<4, 3, 2, 4, G>), grid, dim3(512), 2 * 128 * 256, s, w, a);
        else if (best == 128) hipLaunchKernelGGL((tile_kernel<4, 2, 2, 4, G>), grid, dim3(512), 2 * 128 * 256, s, w, a);
        else hipLaunchKernelGGL((tile_kernel<2, 2, 2, 2, G>), grid, dim3(256), 2 * 64 * 256, s, w, a);
        return;
    }
    int mt = a.m <= 16 ? 1 : a.m <= 32 ? 2 : 4;
    const size_t lds = (size_t)chunks * 4 * mt * 1024;
    // Four tiles a CU and more: 32 x 51866 x 1280 takes 16.2 us by row_kernel, 43.6 by split_kernel (1 row: 9.8, 13.8);
    // 32 x 5120 x 1280 (320 tiles) 12.5 and 7.4. x has to fit into LDS.
    if (tiles >= 4 * cus && lds <= 160 * 1024) {
        const int waves = std::min(16, blocks(tiles, (long)cus * blocks(tiles, 16L * cus)));
        const dim3 grid(blocks(tiles, waves), blocks(a.m, 16 * mt)), block(64 * waves);
        if (mt == 1) hipLaunchKernelGGL((row_kernel<1, G>), grid, block, lds, s, w, a);
        else if (mt == 2) hipLaunchKernelGGL((row_kernel<2, G>), grid, block, lds, s, w, a);
        else hipLaunchKernelGGL((row_kernel<4, G>), grid, block, lds, s, w, a);
        return;
    }
    // Fewer rows of x a workgroup where that leaves CUs without one: 32 x 1280 x 5120 takes 7.3 us with 16 of them, 11.7 with 32.
    while (mt > 1 && (long)tiles * blocks(a.m, 16 * mt) < cus) mt /= 2;
    const int most = mt == 4 ? 8 : 16, waves = blocks(chunks, blocks(chunks, most));
    const dim3 grid(tiles, blocks(a.m, 16 * mt)), block(64 * waves);
    const size_t red = (size_t)waves * 4 * mt * 68 * 4;
    if (mt == 1) hipLaunchKernelGGL((split_kernel<1, G>), grid, block, red, s, w, a);
    else if (mt == 2) hipLaunchKernelGGL((split_kernel<2, G>), grid, block, red, s, w, a);
    else hipLaunchKernelGGL((split_kernel<4, G>), grid, block, red, s, w, a);
}

unsigned entry_groups(const MzW4& w) { return (unsigned)(((long)(w.n + 15) / 16 * (w.k / 128) + 3) / 4); }

}  // namespace

hipError_t mz_w4_pack_launch(hipStream_t s, const MzW4& w, const f16* src, long ld) {
    hipLaunchKernelGGL(pack_kernel, dim3(entry_groups(w)), dim3(256), 0, s, w, src, ld);
    return hipGetLastError();
}

hipError_t mz_w4_unpack_launch(hipStream_t s, const MzW4& w, f16* dst, long ld) {
    hipLaunchKernelGGL(unpack_kernel, dim3(entry_groups(w)), dim3(256), 0, s, w, dst, ld);
    return hipGetLastError();
}

hipError_t mz_w4_linear_launch(hipStream_t s, const MzW4& w, const MzW4Linear& a) {
    if (w.group == 32) linear_launch<4>(s, w, a);
    else if (w.group == 64) linear_launch<2>(s, w, a);
    else linear_launch<1>(s, w, a);
    return hipGetLastError();
}
