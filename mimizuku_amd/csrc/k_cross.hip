// Attention over an encoder's fp16 keys and values of any length (mz_cross_attention_args in mimizuku.h).
#include <algorithm>

#include "mz_common.h"
#include "mz_kernels.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f, NOTHING = -1e30f;

// what a row's queries see: positions first .. end - 1 of its slot
struct Seen {
    long slot;
    int first, end, count;
};
__device__ __forceinline__ Seen seen_of(const MzCross& a, int r) {
    Seen s;
    s.slot = a.slot ? a.slot[r] : r;
    s.count = a.count ? min(max(a.count[r], 0), a.tokens) : a.tokens;
    s.first = a.first ? max(a.first[r], 0) : 0;
    s.end = a.len ? min(max(a.len[r], 0), a.positions) : a.positions;
    if (s.slot < 0 || s.slot >= a.slots) s.slot = s.end = 0;
    s.end = max(s.end, s.first);  // (nothing: first .. first)
    return s;
}

// A wave: one query. 64 positions at a time, a lane a position for the scores and a channel for the sums.
__global__ void __launch_bounds__(64) simple_kernel(MzCross a) {
    __shared__ float qs[64];
    const int lane = threadIdx.x, pair = blockIdx.x, i = blockIdx.y / (a.heads / a.kv_heads);
    const int r = pair / a.kv_heads, kh = pair - r * a.kv_heads, grp = a.heads / a.kv_heads, h = kh * grp + blockIdx.y % grp;
    const Seen s = seen_of(a, r);
    if (i >= s.count) return;
    qs[lane] = (float)a.q[r * a.q_row + i * a.q_token + h * a.q_head + lane];
    __syncthreads();
    const f16* k = a.k + s.slot * a.k_slot + kh * a.k_head;
    const f16* v = a.v + s.slot * a.v_slot + kh * a.v_head;
    const float scale2 = a.scale * LOG2E;
    auto score = [&](int p) {
        float d = 0.f;
        for (int c = 0; c < 64; c += 8) {
            const f16x8 x = ld8(k + p * a.k_pos + c);
            for (int e = 0; e < 8; e++) d = fmaf((float)x[e], qs[c + e], d);
        }
        return d * scale2;
    };
    float m = NOTHING, l = 0.f, o = 0.f;
    for (int p0 = s.first; p0 < s.end; p0 += 64) {
        const int p = p0 + lane;
        const float d = p < s.end ? score(p) : -INFINITY;
        const float mn = fmaxf(m, wave_max(d)), f = __builtin_amdgcn_exp2f(m - mn), x = __builtin_amdgcn_exp2f(d - mn);
        m = mn;
        l = l * f + wave_sum(x);
        o *= f;
        for (int j = 0; j < min(64, s.end - p0); j++)
            o = fmaf(__shfl(x, j), (float)v[(p0 + j) * a.v_pos + lane], o);
    }
    a.out[r * a.out_row + i * a.out_token + h * a.out_head + lane] = (f16)(l == 0.f ? 0.f : o / l);
    const float lse2 = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
    if (a.lse && lane == 0) a.lse[((long)r * a.tokens + i) * a.heads + h] = lse2 * LN2;
    if (!a.align) return;
    const int at = a.head_slot[h];
    bool mine = at >= 0 && at < a.align_heads;
    for (int j = 0; j < h; j++) mine &= a.head_slot[j] != at;
    if (!mine) return;
    float* row = a.align + (((long)r * a.tokens + i) * a.align_heads + at) * a.align_cols;
    for (int p = lane; p < a.align_cols; p += 64)
        row[p] = p >= s.first && p < s.end ? __builtin_amdgcn_exp2f(score(p) - lse2) : 0.f;
}

}  // namespace

bool mz_cross_fits(const MzCross& a) {
    const long nq = (long)a.tokens * (a.heads / a.kv_heads);
    return (long)a.rows * a.kv_heads < (1L << 23) - 8 && nq <= 16L * 65535;
}

size_t mz_cross_work(const MzCross& a) { return 0; }

hipError_t mz_cross_launch(hipStream_t s, const MzCross& a) {
    hipLaunchKernelGGL(simple_kernel, dim3(a.rows * a.kv_heads, a.tokens * (a.heads / a.kv_heads)), dim3(64), 0, s, a);
    return hipGetLastError();
}
