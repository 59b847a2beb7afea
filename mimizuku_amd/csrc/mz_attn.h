// What the two attentions over keys and values in memory share (8-bit caches, an encoder's output): a wave's softmax state lies
// in the results of 16x16 products, a query a column.
#pragma once
#include "mz_common.h"

namespace {

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

// (the median of two numbers and infinity is the larger one. A maximum would make each operand quiet first, and so would a
// median with an infinity that the compiler knows.)
__device__ __forceinline__ float larger(float a, float b, float inf) { return __builtin_amdgcn_fmed3f(a, b, inf); }

// x / d for x below 2^31 by r = min(2^32 / d, 2^32 - 1): no more than one too small before the correction (a division by a
// number not known beforehand takes about twenty dependent instructions)
__device__ __forceinline__ int divided(int x, int d, unsigned r) {
    const int q = (int)__umulhi((unsigned)x, r);
    return q + ((q + 1) * (long)d <= x);
}
constexpr int STATE = 66;  // floats of a query's partial state: 64 channels, maximum, sum

// Alignment indices of the query heads h0 .. h0 + n - 1, by all threads of the workgroup: of heads with one index the
// first has it. mine: head_slot[threadIdx.x], requested earlier.
template <int THREADS>
__device__ __forceinline__ void align_indices(const int* head_slot, int align_heads, int h0, int n, int mine, int (&index)[64]) {
    __shared__ int slots[64];
    const int tid = threadIdx.x;
    for (int j = tid; j < h0 + n; j += THREADS) {
        const int s = j == tid ? mine : head_slot[j];
        if (j >= h0) slots[j - h0] = index[j - h0] = s < align_heads ? s : -1;
    }
    __syncthreads();
    for (int j = tid; j < h0 + n; j += THREADS) {
        const int s = j == tid ? mine : head_slot[j];
        for (int k = max(0, j - h0 + 1); k < n; k++)
            if (slots[k] == s) index[k] = -1;
    }
    __syncthreads();
}

}  // namespace
