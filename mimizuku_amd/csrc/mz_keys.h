// Logits with their ids as numbers in one order, and networks that put them in it within a wave (token scores, the next token).
#pragma once
#include "mz_common.h"

namespace {

// A value and an id as one number: the larger the better, of equal values (-0 is +0) the lowest id; 0: none (below -inf with
// any id).
// 62 bits, so that as a number of 64 bits it is positive, finite and in the same order, and v_max_f64 takes the larger one.
typedef unsigned long long Key;
constexpr unsigned IDS = 1u << 30;
__device__ __forceinline__ Key key_of(float v, int id) {
    const unsigned u = __builtin_bit_cast(unsigned, v + 0.f);  // (a sum of zeros is +0 unless both are -0)
    return (Key)(u ^ ((unsigned)((int)u >> 31) | 0x80000000u)) << 30 | (IDS - 1 - (unsigned)id);
}
__device__ __forceinline__ float value_of(Key k) {
    const unsigned u = (unsigned)(k >> 30);
    return k ? __builtin_bit_cast(float, u ^ (~(unsigned)((int)u >> 31) | 0x80000000u)) : -INFINITY;
}
__device__ __forceinline__ int id_of(Key k) { return (int)(IDS - 1 - ((unsigned)k & (IDS - 1))); }
// (through the compiler each operand would be made quiet first, another such instruction each; the two wait states are those
// that a DPP or lane-swap reader of a vector result needs, which the compiler does not see here)
__device__ __forceinline__ Key larger(Key a, Key b) {
    Key r;
    asm("v_max_f64 %0, %1, %2\n\ts_nop 1" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ Key smaller(Key a, Key b) {
    Key r;
    asm("v_min_f64 %0, %1, %2\n\ts_nop 1" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ Key lane_key(Key k, int i) {
    return (Key)(unsigned)__builtin_amdgcn_readlane((int)(k >> 32), i) << 32 | (unsigned)__builtin_amdgcn_readlane((int)k, i);
}
// ---- keys in order: networks of compare-and-exchange steps across lanes, best first within each row of 16 lanes. A step is
// six instructions or so; finding the best of 64 lanes k times over takes about 70 dependent ones each time.
template <int CTRL>
__device__ __forceinline__ Key moved(Key k) {
    return (Key)(unsigned)dpp_i<CTRL>((int)(k >> 32)) << 32 | (unsigned)dpp_i<CTRL>((int)k);
}
__device__ __forceinline__ int xor4(int v) {  // lanes with bit 2 clear read 4 on, the others 4 back
    const int t = __builtin_amdgcn_update_dpp(0, v, 0x104, 0xF, 0x5, false);
    return __builtin_amdgcn_update_dpp(t, v, 0x114, 0xF, 0xA, false);
}
// the better of k and p where `first` is set, the other one elsewhere
__device__ __forceinline__ Key step(Key k, Key p, bool first) {
    const Key a = larger(k, p), b = smaller(k, p);  // (both, where a branch would be taken)
    return first ? a : b;
}
// a row whose better half is anywhere in bitonic order, best first
__device__ __forceinline__ Key cleaned(Key k, int lane) {
    k = step(k, moved<0x128>(k), !(lane & 8));
    k = step(k, (Key)(unsigned)xor4((int)(k >> 32)) << 32 | (unsigned)xor4((int)k), !(lane & 4));
    k = step(k, moved<0x4E>(k), !(lane & 2));
    return step(k, moved<0xB1>(k), !(lane & 1));
}
__device__ __forceinline__ Key other_row(Key k, int lane) {
    const auto h = __builtin_amdgcn_permlane16_swap((unsigned)(k >> 32), (unsigned)(k >> 32), false, false);
    const auto l = __builtin_amdgcn_permlane16_swap((unsigned)k, (unsigned)k, false, false);
    return lane & 16 ? (Key)(unsigned)h[0] << 32 | (unsigned)l[0] : (Key)(unsigned)h[1] << 32 | (unsigned)l[1];
}
__device__ __forceinline__ Key other_half(Key k, int lane) {
    const auto h = __builtin_amdgcn_permlane32_swap((unsigned)(k >> 32), (unsigned)(k >> 32), false, false);
    const auto l = __builtin_amdgcn_permlane32_swap((unsigned)k, (unsigned)k, false, false);
    return lane & 32 ? (Key)(unsigned)h[0] << 32 | (unsigned)l[0] : (Key)(unsigned)h[1] << 32 | (unsigned)l[1];
}
// each row of 16 lanes in order, best first
__device__ __forceinline__ Key sorted_rows(Key k, int lane) {
    k = step(k, moved<0xB1>(k), !(lane & 1));
    k = step(k, moved<0x1B>(k), !(lane & 2));
    k = step(k, moved<0xB1>(k), !(lane & 1));
    k = step(k, moved<0x141>(k), !(lane & 4));
    k = step(k, moved<0x4E>(k), !(lane & 2));
    k = step(k, moved<0xB1>(k), !(lane & 1));
    k = step(k, moved<0x140>(k), !(lane & 8));
    k = step(k, (Key)(unsigned)xor4((int)(k >> 32)) << 32 | (unsigned)xor4((int)k), !(lane & 4));
    k = step(k, moved<0x4E>(k), !(lane & 2));
    k = step(k, moved<0xB1>(k), !(lane & 1));
    return k;
}

}  // namespace
