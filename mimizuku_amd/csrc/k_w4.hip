// Products with 4-bit weights (mz_w4 in mimizuku.h).
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
    // row i is row 4 (i / 4) + i % 4: place [i / 4][group][i % 4]
    const int groups = 128 / w.group;
    if (j == 0)
#pragma unroll
        for (int s = 0; s < 4; s++)
            if (s % words == 0) w.scales[(entry * 4 + (i >> 2)) * groups * 4 + s / words * 4 + (i & 3)] = scale[s];
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
        const float d = (float)w.scales[(entry * 4 + (i >> 2)) * groups * 4 + s / words * 4 + (i & 3)];
        f16x8 y;
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = (f16)((float)((int)(q[s] >> bit_of(e) & 15) - 8) * d);
        *(f16x8*)(dst + (t * 16 + i) * ld + c * 128 + 32 * s + 8 * j) = y;
    }
}

// A thread: one output of a tile of 16 rows of weights x 16 rows of x.
__global__ void __launch_bounds__(256) linear_kernel(MzW4 w, MzW4Linear a) {
    const int i = threadIdx.x & 15, mi = blockIdx.y * 16 + (threadIdx.x >> 4), chunks = w.k / 128, groups = 128 / w.group;
    const long t = blockIdx.x, n = t * 16 + i;
    if (mi >= a.m || n >= w.n) return;
    const f16* x = a.x + mi * a.ldx;
    float sum = 0.f;
    for (int c = 0; c < chunks; c++) {
        const long entry = t * chunks + c;
        for (int g = 0; g < groups; g++) {
            float part = 0.f;
            for (int k = g * w.group; k < (g + 1) * w.group; k += 8) {
                const int s = k / 32, j = k / 8 % 4;
                const unsigned q = *(const unsigned*)(w.codes + (entry * 64 + 16 * j + i) * 16 + 4 * s);
                const f16x8 v = ld8(x + c * 128 + k);
                for (int e = 0; e < 8; e++) part = fmaf((float)((int)(q >> bit_of(e) & 15) - 8), (float)v[e], part);
            }
            sum = fmaf((float)w.scales[(entry * 4 + (i >> 2)) * groups * 4 + g * 4 + (i & 3)], part, sum);
        }
    }
    if (a.bias) sum += (float)a.bias[n];
    const long o = mi * a.ldo + n;
    switch (a.epilogue) {
        case 0: ((f16*)a.out)[o] = (f16)sum; break;
        case 1: ((f16*)a.out)[o] = (f16)gelu_erf_h(sum); break;
        case 2: ((float*)a.out)[o] += sum; break;
        default: ((float*)a.out)[o] = sum;
    }
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
    hipLaunchKernelGGL(linear_kernel, dim3((w.n + 15) / 16, (a.m + 15) / 16), dim3(256), 0, s, w, a);
    return hipGetLastError();
}
