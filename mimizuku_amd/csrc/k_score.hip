// Token scores (mz_score_args in mimizuku.h): log probability of a given token, entropy and best alternatives of rows of
// logits, in one pass over them.
//
// With m a row's maximum, at element i0, S the sum of exp(x - m) over the others and U that of exp(x - m)(x - m):
// ln sum exp x = m + log1p(S), log p = (x - m) - log1p(S), entropy = log1p(S) - U / (1 + S). The last two terms are both
// positive and S does not hold the 1 of the maximum, so that sure rows (S far below 1) keep their digits.
#include <algorithm>

#include "mz_common.h"
#include "mz_kernels.h"

namespace {

constexpr int PER_LANE = 16, CHUNK = 64 * PER_LANE;  // elements that a lane / a wave holds at a time
constexpr int PARTS = 64;                            // most waves that share a row: one lane each where they are joined
constexpr int NONE = 0x7fffffff;
constexpr float LOG2E = 1.4426950408889634f;

// what one wave knows of its elements
struct Part {
    float m, s, u, pad;
    float v[MZ_SCORE_ALTS];  // its best alternatives, best first
    int id[MZ_SCORE_ALTS];
};

// d = x - m to exp(d) and exp(d) d, 0 and 0 for -inf
__device__ __forceinline__ void add(float x, float m, float& s, float& u) {
    const float d = x - m, e = __builtin_amdgcn_exp2f(d * LOG2E);
    s += e;
    u = fmaf(e, fmaxf(d, -200.f), u);
}

// Lane i < parts holds part i: the row's results. The alternatives are taken one after the other from the parts' lists.
template <typename T>
__device__ __forceinline__ void finish(const MzScores& p, int r, const Part* part, int parts, int lane) {
    const long n = p.at ? (long)*p.at + p.at_add : 0;
    if (n < 0 || n >= p.out_stride) return;
    const bool on = lane < parts;
    float mi = on ? part[lane].m : -INFINITY;
    const float si = on ? part[lane].s : 0.f, ui = on ? part[lane].u : 0.f;
    const float m = wave_max(mi);
    // one of the parts with the row's maximum holds the element that S leaves out; the others' maxima count in it
    const bool owner = lane == __ffsll((unsigned long long)__ballot(mi == m)) - 1;
    const float d = mi - m, e = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(d * LOG2E);
    const float t = si + 1.f;
    // (a part of NaN only has m -inf and s NaN)
    const float S = wave_sum(owner || si != si ? si : t * e), U = wave_sum(owner ? ui : e == 0.f ? 0.f : e * fmaf(t, d, ui));
    const bool bad = S != S || m == INFINITY;
    const float z = log1pf(S);
    const long o = r * p.out_stride + n;
    if (lane == 0 && p.logp) {
        const int tok = n < p.token_stride ? p.tokens[r * p.token_stride + n] : -1;
        float lp = 0.f;
        if (tok >= 0) {
            if (bad || tok >= p.vocab) lp = NAN;
            else if (m == -INFINITY || (p.mask && p.mask[tok])) lp = -INFINITY;
            else lp = ((float)((const T*)p.logits)[r * p.ld + tok] - m) - z;
        }
        p.logp[o] = lp;
    }
    if (lane == 0 && p.entropy) p.entropy[o] = bad ? NAN : m == -INFINITY ? 0.f : z - U / (1.f + S);
    float v = on && p.alts ? part[lane].v[0] : -INFINITY;
    int id = on && p.alts ? part[lane].id[0] : NONE, at = 0;
    for (int k = 0; k < p.alts; k++) {
        float bv = v;
        int bi = id;
        wave_argmax(bv, bi);
        if (lane == 0) {
            if (p.alt_ids) p.alt_ids[o * p.alts + k] = bad || bv == -INFINITY ? -1 : bi;
            if (p.alt_logp) p.alt_logp[o * p.alts + k] = bad ? NAN : bv == -INFINITY ? -INFINITY : (bv - m) - z;
        }
        if (id == bi && v == bv && v > -INFINITY) {
            at++;
            v = at < p.alts ? part[lane].v[at] : -INFINITY;
            id = at < p.alts ? part[lane].id[at] : NONE;
        }
    }
}

// A workgroup's share of a row, four waves taking chunks of 1024 elements in turn. `splits` workgroups share a row, each
// wave writing its part to the workspace (to LDS and the row finished here where there is one).
template <typename T, bool MASK>
__global__ void __launch_bounds__(256) score_kernel(MzScores p, int splits) {
    constexpr int V = 16 / sizeof(T), G = PER_LANE / V;  // elements of a 16-byte load, loads of a chunk
    typedef T TV __attribute__((ext_vector_type(V)));
    __shared__ Part lds[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = blockIdx.x / splits, split = blockIdx.x - r * splits;
    const T* row = (const T*)p.logits + r * p.ld;
    // the row's 16-byte pieces, the first of which begins `off` elements before it
    const int off = (int)((uintptr_t)row % 16 / sizeof(T));
    const int chunks = (p.vocab + off + CHUNK - 1) / CHUNK, share = (chunks + splits - 1) / splits;
    const int c0 = split * share, c1 = min(c0 + share, chunks);

    struct Raw {
        TV x[G];
        unsigned char mask[PER_LANE];
    };
    auto first = [&](int c, int j) { return (c * G + j) * 64 * V + lane * V - off; };  // id of lane's element 0 of load j
    auto fetch = [&](int c, Raw& w) {
#pragma unroll
        for (int j = 0; j < G; j++) {
            const int e = first(c, j);
            if (e >= 0 && e + V <= p.vocab) {
                w.x[j] = __builtin_nontemporal_load((const TV*)(row + e));
                if (MASK) __builtin_memcpy(w.mask + j * V, p.mask + e, V);
            } else {
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const bool in = e + k >= 0 && e + k < p.vocab;
                    w.x[j][k] = in ? row[e + k] : (T)-INFINITY;
                    if (MASK) w.mask[j * V + k] = in ? p.mask[e + k] : 0;
                }
            }
        }
    };

    float m = -INFINITY, S = 0.f, U = 0.f;  // m of the wave, the sums of the lane
    float lv = -INFINITY, thr = -INFINITY;  // lane k: alternative k; thr: the last one's value
    int li = NONE;
    auto chunk = [&](int c, const Raw& w) {
        float x[PER_LANE], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < PER_LANE; j++) {
            x[j] = (float)w.x[j / V][j % V];
            if (MASK) x[j] = w.mask[j] ? -INFINITY : x[j];
            top = fmaxf(top, x[j]);
        }
        const unsigned long long up = __ballot(top > m);
        if (up) {  // a new maximum: the sums so far, the old maximum among them, become multiples of it
            const float mn = wave_max(top);
            const bool own = lane == __ffsll((unsigned long long)__ballot(top == mn)) - 1;
            if (m > -INFINITY) {
                const float d = m - mn, f = __builtin_amdgcn_exp2f(d * LOG2E);
                const float t = S + (lane == 0 ? 1.f : 0.f);
                U = f == 0.f ? 0.f * U : f * fmaf(t, d, U);
                S = t * f;
            }
            m = mn;
            bool left = own;  // one element of the maximum is left out
#pragma unroll
            for (int j = 0; j < PER_LANE; j++) {
                const bool out = left && x[j] == mn;
                left = left && !out;
                if (!out) add(x[j], m, S, U);
            }
        } else {
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int j = 0; j < PER_LANE; j++) add(x[j], ref, S, U);
        }
        if (p.alts)
            while (__ballot(top > thr)) {
                // the chunk's best, lowest id first, into its place of the list
                int bi = NONE;
#pragma unroll
                for (int j = PER_LANE - 1; j >= 0; j--)
                    if (x[j] == top) bi = first(c, j / V) + j % V;
                float bv = top;
                int id = bi;
                wave_argmax(bv, id);
                const int at = __popcll(__ballot(lane < p.alts && (lv > bv || (lv == bv && li < id))));
                const float pv = dpp_f<0x111>(lv);  // the lane before
                const int pi = dpp_i<0x111>(li);
                if (lane < p.alts && lane >= at) {
                    lv = lane == at ? bv : pv;
                    li = lane == at ? id : pi;
                }
                thr = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, lv), p.alts - 1));
                if (bi == id) {
                    top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < PER_LANE; j++) {
                        if (first(c, j / V) + j % V == id) x[j] = -INFINITY;
                        top = fmaxf(top, x[j]);
                    }
                }
            }
    };
    Raw w0, w1;
    int c = c0 + wave;
    if (c < c1) fetch(c, w0);
    for (; c < c1; c += 8) {
        if (c + 4 < c1) fetch(c + 4, w1);
        chunk(c, w0);
        if (c + 4 < c1) {
            if (c + 8 < c1) fetch(c + 8, w0);
            chunk(c + 4, w1);
        }
    }
    S = wave_sum(S);
    U = wave_sum(U);
    Part* part = splits > 1 ? (Part*)p.work + ((long)r * splits + split) * 4 + wave : lds + wave;
    if (lane == 0) {
        part->m = m;
        part->s = S;
        part->u = U;
    }
    if (lane < p.alts) {
        part->v[lane] = lv;
        part->id[lane] = li;
    }
    if (splits > 1) return;
    __syncthreads();
    if (wave == 0) finish<T>(p, r, lds, 4, lane);
}

template <typename T>
__global__ void __launch_bounds__(64) score_join_kernel(MzScores p, int parts) {
    finish<T>(p, blockIdx.x, (const Part*)p.work + (long)blockIdx.x * parts, parts, threadIdx.x);
}

int score_splits(const MzScores& p) {
    const long chunks = (p.vocab + CHUNK - 1) / CHUNK, want = 4L * mz_cu_count() / p.rows;
    return (int)std::max(1L, std::min({want, (chunks + 3) / 4, (long)PARTS / 4}));
}

template <typename T>
hipError_t launch(hipStream_t s, const MzScores& p) {
    const int splits = score_splits(p);
    const dim3 grid((long)p.rows * splits);
    if (p.mask) hipLaunchKernelGGL((score_kernel<T, true>), grid, dim3(256), 0, s, p, splits);
    else hipLaunchKernelGGL((score_kernel<T, false>), grid, dim3(256), 0, s, p, splits);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || splits == 1) return e;
    hipLaunchKernelGGL(score_join_kernel<T>, dim3(p.rows), dim3(64), 0, s, p, 4 * splits);
    return hipGetLastError();
}

}  // namespace

size_t mz_scores_work(const MzScores& p) {
    const int splits = score_splits(p);
    return splits > 1 ? (size_t)p.rows * splits * 4 * sizeof(Part) : 0;
}

hipError_t mz_scores_launch(hipStream_t s, const MzScores& p) { return p.half ? launch<f16>(s, p) : launch<float>(s, p); }
