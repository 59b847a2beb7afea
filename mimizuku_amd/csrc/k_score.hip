// Token scores (mz_score_args in mimizuku.h): log probability of a given token, entropy and best alternatives of rows of
// logits. Plain kernel: one workgroup per row, one pass for the maximum, one for the sums, one per alternative.
#include "mz_common.h"
#include "mz_kernels.h"

namespace {

// S = sum over all elements but the (first) largest of exp(x - m), T = the same sum of exp(x - m)(x - m): then
// ln sum exp x = m + log1p(S) and the entropy is log1p(S) - T / (1 + S), both terms positive, so that a sure row's log
// probability and entropy keep their digits.
template <typename T>
__global__ void __launch_bounds__(256) score_kernel(MzScores p) {
    __shared__ float sv[4];
    __shared__ int si[4];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long n = p.at ? (long)*p.at + p.at_add : 0;
    if (n < 0 || n >= p.out_stride) return;
    const T* x = (const T*)p.logits + r * p.ld;
    auto get = [&](int i) { return p.mask && p.mask[i] ? -INFINITY : (float)x[i]; };
    auto sum = [&](float v) {
        v = wave_sum(v);
        __syncthreads();
        if (lane == 0) sv[wave] = v;
        __syncthreads();
        return (sv[0] + sv[1]) + (sv[2] + sv[3]);
    };
    // the best (value, id) behind (after, id0) in the order of alternatives
    auto next = [&](float after, int id0, float& v, int& id) {
        v = -INFINITY;
        id = 0x7fffffff;
        for (int i = tid; i < p.vocab; i += 256) {
            const float y = get(i);
            if ((y < after || (y == after && i > id0)) && (y > v || (y == v && i < id))) {
                v = y;
                id = i;
            }
        }
        wave_argmax(v, id);
        __syncthreads();
        if (lane == 0) {
            sv[wave] = v;
            si[wave] = id;
        }
        __syncthreads();
        v = sv[0];
        id = si[0];
        for (int w = 1; w < 4; w++)
            if (sv[w] > v || (sv[w] == v && si[w] < id)) {
                v = sv[w];
                id = si[w];
            }
    };
    float m, v;
    int im, id;
    next(INFINITY, -1, m, im);
    const float m0 = m == -INFINITY ? 0.f : m;
    float S = 0.f, U = 0.f;
    for (int i = tid; i < p.vocab; i += 256) {
        if (i == im) continue;
        const float d = get(i) - m0, e = expf(d);
        S += e;
        U = fmaf(e, fmaxf(d, -200.f), U);
    }
    S = sum(S);
    U = sum(U);
    const bool bad = S != S || m == INFINITY;
    const float z = log1pf(S);
    const long o = r * p.out_stride + n;
    if (tid == 0 && p.logp) {
        const int t = n < p.token_stride ? p.tokens[r * p.token_stride + n] : -1;
        p.logp[o] = t < 0 ? 0.f : bad || t >= p.vocab ? NAN : m == -INFINITY ? -INFINITY : get(t) - m - z;
    }
    if (tid == 0 && p.entropy) p.entropy[o] = bad ? NAN : m == -INFINITY ? 0.f : z - U / (1.f + S);
    v = INFINITY;
    id = -1;
    for (int k = 0; k < p.alts; k++) {
        if (id != 0x7fffffff) next(v, id, v, id);
        if (v == -INFINITY) id = 0x7fffffff;
        if (tid == 0) {
            if (p.alt_ids) p.alt_ids[o * p.alts + k] = bad || id == 0x7fffffff ? -1 : id;
            if (p.alt_logp) p.alt_logp[o * p.alts + k] = bad ? NAN : id == 0x7fffffff ? -INFINITY : v - m - z;
        }
    }
}

}  // namespace

size_t mz_scores_work(const MzScores&) { return 0; }

hipError_t mz_scores_launch(hipStream_t s, const MzScores& p) {
    if (p.half) hipLaunchKernelGGL(score_kernel<f16>, dim3(p.rows), dim3(256), 0, s, p);
    else hipLaunchKernelGGL(score_kernel<float>, dim3(p.rows), dim3(256), 0, s, p);
    return hipGetLastError();
}
