// The next token of rows of logits (mz_sample_args in mimizuku.h).
//
// The kept tokens are the first ones in the order of falling logits, of equal ones the lower id first: those with a logit above
// some value, and of those with that value the ids up to some id. So the limits are each a pair (value, id), the kept set is
// above the highest of them, and no row is sorted.
//
// Weights are whole multiples of 2^-shift: sums of them are exact in 64 bits whatever their order.
#include <algorithm>

#include "mz_common.h"
#include "mz_kernels.h"

namespace {

typedef unsigned long long u64;

// a logit as a number in the same order, -0 and +0 alike, -inf the lowest
__device__ __forceinline__ unsigned key_of(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v + 0.f);
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
constexpr unsigned LOWEST = 0x007fffffu;  // key of -inf

constexpr int THREADS = 256;

template <typename T, typename F>
__device__ T block_reduce(T v, F f) {
    __shared__ T part[THREADS];
    __syncthreads();
    part[threadIdx.x] = v;
    __syncthreads();
    for (int o = THREADS / 2; o; o /= 2) {
        if ((int)threadIdx.x < o) part[threadIdx.x] = f(part[threadIdx.x], part[threadIdx.x + o]);
        __syncthreads();
    }
    return part[0];
}
template <typename T>
__device__ T block_sum(T v) {
    return block_reduce(v, [](T a, T b) { return a + b; });
}

__global__ void __launch_bounds__(THREADS) simple_kernel(MzSample a, int shift) {
    const long r = blockIdx.x;
    const int n = a.at ? *a.at + a.at_add : 0, tid = threadIdx.x;
    if (n < 0 || n >= a.stride) return;
    const long at = r * a.stride + n;
    auto get = [&](int i) -> float {
        if (a.mask && a.mask[i]) return -INFINITY;
        return a.half ? (float)((const f16*)a.logits)[r * a.ld + i] : ((const float*)a.logits)[r * a.ld + i];
    };
    float top = -INFINITY;
    int bad = 0, count = 0;
    for (int i = tid; i < a.vocab; i += THREADS) {
        const float x = get(i);
        bad |= !(x < INFINITY);
        count += x > -INFINITY;
        top = fmaxf(top, x);
    }
    top = block_reduce(top, [](float x, float y) { return fmaxf(x, y); });
    bad = block_sum(bad);
    count = block_sum(count);
    const float t = a.temperatures ? a.temperatures[r] : a.temperature, top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    const float min_p = a.min_ps ? a.min_ps[r] : a.min_p;
    const int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    bad |= !(t >= 0.f) || t == INFINITY || top_p != top_p || min_p != min_p;
    if (bad || !count) {
        if (tid == 0) {
            a.tokens[at] = -1;
            if (a.logp) a.logp[at] = bad ? NAN : -INFINITY;
            if (a.kept) a.kept[at] = 0;
        }
        return;
    }
    const double per = 1.0 / (t > 0.f ? (double)t : 1.0);
    auto weight = [&](float x) -> u64 {
        return x == -INFINITY ? 0 : (u64)rint(ldexp(exp(((double)x - (double)top) * per), shift));
    };
    // kept: key > cut, or key == cut and id <= last
    unsigned cut = LOWEST + 1;
    int last = a.vocab;
    auto in = [&](float x, int i) {
        const unsigned k = key_of(x);
        return k > cut || (k == cut && i <= last);
    };
    // the highest key that f, a number falling with rising keys, is at least `need` for
    auto highest = [&](auto f, auto need) {
        unsigned k = 0;
        for (unsigned b = 1u << 31; b; b >>= 1)
            if (f(k | b) >= need) k |= b;
        return k;
    };
    // the id of the need-th token with that key
    auto nth = [&](unsigned k, int need) {
        int lo = 0, hi = a.vocab - 1;
        while (lo < hi) {
            const int mid = lo + (hi - lo) / 2;
            int c = 0;
            for (int i = tid; i <= mid; i += THREADS) c += key_of(get(i)) == k;
            if (block_sum(c) >= need) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    };
    const int k_limit = t == 0.f ? 1 : top_k > 0 ? top_k : a.vocab;
    if (k_limit < count) {
        auto above = [&](unsigned k) {
            int c = 0;
            for (int i = tid; i < a.vocab; i += THREADS) c += key_of(get(i)) >= k;
            return block_sum(c);
        };
        const unsigned k = highest(above, k_limit);
        const int need = k_limit - (k == ~0u ? 0 : above(k + 1));
        cut = k;
        last = nth(k, need);
    }
    if (top_p < 1.f) {
        auto above = [&](unsigned k) {
            u64 s = 0;
            for (int i = tid; i < a.vocab; i += THREADS) {
                const float x = get(i);
                if (key_of(x) >= k && in(x, i)) s += weight(x);
            }
            return block_sum(s);
        };
        const double need = (double)fmaxf(top_p, 0.f) * (double)above(0);
        const unsigned top_key = key_of(top);
        unsigned k = min(highest([&](unsigned x) { return x > top_key ? -1.0 : (double)above(x); }, need), top_key);
        u64 over = above(k + 1);
        float x = __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
        const u64 w = weight(x);
        int c = 1;
        while ((double)(over + c * w) < need && c < a.vocab) c++;
        const int id = nth(k, c);
        if (k > cut || (k == cut && id < last)) {
            cut = k;
            last = id;
        }
    }
    const double low = (double)top + (double)t * log(fmin((double)min_p, 1.0));
    int c = 0;
    u64 s = 0;
    auto kept = [&](float x, int i) { return in(x, i) && (!(min_p > 0.f) || (double)x >= low); };
    for (int i = tid; i < a.vocab; i += THREADS) {
        const float x = get(i);
        if (!kept(x, i)) continue;
        c++;
        s += weight(x);
    }
    c = block_sum(c);
    s = block_sum(s);
    const float u0 = a.u[at], u = u0 >= 0.f ? fminf(u0, 0x1.fffffep-1f) : 0.f;
    const double need = (double)u * (double)s;
    int lo = 0, hi = a.vocab - 1;
    while (lo < hi) {  // the lowest id up to which the weights are more
        const int mid = lo + (hi - lo) / 2;
        u64 run = 0;
        for (int i = tid; i <= mid; i += THREADS) {
            const float x = get(i);
            if (kept(x, i)) run += weight(x);
        }
        if ((double)block_sum(run) > need) hi = mid;
        else lo = mid + 1;
    }
    if (tid == 0) {
        a.tokens[at] = lo;
        if (a.logp) a.logp[at] = (float)(((double)get(lo) - (double)top) * per - log(ldexp((double)s, -shift)));
        if (a.kept) a.kept[at] = c;
    }
}

// weights are multiples of 2^-shift: a row's sum stays below 2^62, and a weight has at most 52 bits
int shift_of(int vocab) {
    int bits = 0;
    while ((1L << bits) < vocab) bits++;
    return std::min(51, 62 - bits);
}

}  // namespace

size_t mz_sample_work(const MzSample& p) { return 0; }

hipError_t mz_sample_launch(hipStream_t s, const MzSample& p) {
    hipLaunchKernelGGL(simple_kernel, dim3(p.rows), dim3(THREADS), 0, s, p, shift_of(p.vocab));
    return hipGetLastError();
}
