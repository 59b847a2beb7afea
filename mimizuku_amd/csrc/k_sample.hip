// The next token of rows of logits (mz_sample_args in mimizuku.h).
//
// The kept tokens are the first ones in the order of falling logits, of equal ones the lower id first: those with a logit above
// some value, and of those with that value the ids up to some id. So each limit is a pair (value, id), the kept set is what
// passes the highest of them, and no row is sorted. Where a limit lies is found by sums over intervals of values, the one that
// holds it taken apart again.
//
// Weights are whole multiples of 2^-shift: sums of them are exact in 64 bits whatever their order.
//
// A workgroup of 1024 threads takes a row and reads it again for each pass. Limits leave few tokens of most rows: those that the limits can reach go into a list, and up to 64 of them are put in order by one wave.
#include <algorithm>

#include "mz_common.h"
#include "mz_keys.h"
#include "mz_kernels.h"

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int BINS = THREADS, BIN_BITS = 10, LIST = THREADS;

// a logit as a number in the opposite order, -0 and +0 alike
__device__ __forceinline__ unsigned order_of(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v + 0.f);
    return u ^ (~(unsigned)((int)u >> 31) & 0x7fffffffu);
}
__device__ __forceinline__ float value_at(unsigned o) { return __builtin_bit_cast(float, o ^ (~(unsigned)((int)o >> 31) & 0x7fffffffu)); }

// exp((x - top) / t) in steps of 2^-shift, 0 for -inf. With s = (x - top) / (t ln 2), n the whole number next to it and f = s - n:
// n is in the low bits of s + 1.5 * 2^52, 2^f is a polynomial of degree 8 through its values at nine Chebyshev nodes (relative
// error below 1.1e-12), 2^n goes into its exponent, and the sum with 2^52 has the result, rounded, in its low 52 bits.
struct Weights {
    double top, per;  // per: 1 / (t ln 2)
    double lowest;    // -200 / per: what is further below the top has weight 0
    int shift;
    __device__ __forceinline__ u64 operator()(float x) const {
        const double d = fmax((double)x - top, lowest), s = fma(d, per, 0x1.8p52), f = fma(d, per, 0x1.8p52 - s);
        double p = 0x1.63d136366db24p-20;
        p = fma(p, f, 0x1.00dc4a532fb8ep-16);
        p = fma(p, f, 0x1.4308ac85aa947p-13);
        p = fma(p, f, 0x1.5d8745a728441p-10);
        p = fma(p, f, 0x1.3b2ab7181b755p-7);
        p = fma(p, f, 0x1.c6b08dd6fd234p-5);
        p = fma(p, f, 0x1.ebfbdff823cedp-3);
        p = fma(p, f, 0x1.62e42fef84cf0p-1);
        p = fma(p, f, 1.0);
        const u64 bits = __builtin_bit_cast(u64, p) + ((u64)(__builtin_bit_cast(u64, s) + shift) << 52);
        return __builtin_bit_cast(u64, __builtin_bit_cast(double, bits) + 0x1p52) & ((1ULL << 52) - 1);
    }
};

// ---------------------------------------------------------------- sums over a workgroup

struct Add {
    template <typename T>
    __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct Min {
    template <typename T>
    __device__ __forceinline__ T operator()(T a, T b) const { return b < a ? b : a; }
};
struct Max {
    template <typename T>
    __device__ __forceinline__ T operator()(T a, T b) const { return b > a ? b : a; }
};
template <int CTRL, typename T>
__device__ __forceinline__ T moved_of(T v) {
    if constexpr (sizeof(T) == 8) return __builtin_bit_cast(T, moved<CTRL>(__builtin_bit_cast(u64, v)));
    else return __builtin_bit_cast(T, dpp_i<CTRL>(__builtin_bit_cast(int, v)));
}
template <typename T>
__device__ __forceinline__ T lane_of(T v, int lane) {
    if constexpr (sizeof(T) == 8) return __builtin_bit_cast(T, lane_key(__builtin_bit_cast(u64, v), lane));
    else return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
// f over each aligned 16 lanes, in each of them
template <typename T, typename F>
__device__ __forceinline__ T row_all(T v, F f) {
    v = f(v, moved_of<0xB1>(v));
    v = f(v, moved_of<0x4E>(v));
    v = f(v, moved_of<0x141>(v));
    return f(v, moved_of<0x140>(v));
}
// f over all threads, in every thread
template <typename T, typename F>
__device__ __forceinline__ T block_all(T v, F f) {
    static_assert(WAVES == 16);
    __shared__ T part[WAVES];
    v = row_all(v, f);
    v = f(f(lane_of(v, 0), lane_of(v, 16)), f(lane_of(v, 32), lane_of(v, 48)));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return row_all(part[threadIdx.x & 15], f);
}
// the sum up to and with this lane's: within rows of 16 lanes by 1, 2, 4 and 8, then row 0's last into row 1 and row 2's into row
// 3, then row 1's last into both
__device__ __forceinline__ u64 wave_running(u64 v) {
    auto step = [&](auto lo_hi) {
        v += (u64)(unsigned)lo_hi((int)(v >> 32)) << 32 | (unsigned)lo_hi((int)v);
    };
    step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true); });
    step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true); });
    step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true); });
    step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true); });
    step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false); });
    step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false); });
    return v;
}

// the wave's keys in order, best first
__device__ __forceinline__ Key sorted_wave(Key k, int lane) {
    k = sorted_rows(k, lane);
    k = cleaned(step(k, moved<0x140>(other_row(k, lane)), !(lane & 16)), lane);
    k = step(k, moved<0x140>(other_row(other_half(k, lane), lane)), !(lane & 32));
    k = step(k, other_row(k, lane), !(lane & 16));
    return cleaned(k, lane);
}

// A row's tokens, read again by each pass (from the caches, after the first).
template <typename T, bool MASK>
struct Row {
    static constexpr int V = 16 / sizeof(T);
    typedef T TV __attribute__((ext_vector_type(V)));
    typedef TV __attribute__((aligned(sizeof(T)))) Loaded;
    typedef unsigned Bits __attribute__((aligned(1)));
    struct Piece {
        TV raw;
        unsigned bits[MASK ? V / 4 : 1];
    };
    const T* row;
    const unsigned char* mask;
    int vocab, off, pieces;  // 16-byte pieces of memory; the first begins `off` elements before the row
    int rounds;              // pieces of a thread

    __device__ __forceinline__ void open(const MzSample& a, long r) {
        row = (const T*)a.logits + r * a.ld;
        mask = a.mask;
        vocab = a.vocab;
        off = (int)((uintptr_t)row % 16 / sizeof(T));
        pieces = (vocab + off + V - 1) / V;
        rounds = (pieces + THREADS - 1) / THREADS;
    }
    // where piece p's elements begin, and where they are read: pieces at the row's ends are moved into it
    __device__ __forceinline__ int begin(int p) const { return p * V - off; }
    __device__ __forceinline__ int from(int p) const { return max(min(begin(p), vocab - V), 0); }
    __device__ __forceinline__ int piece(int j) const { return min(j * THREADS + (int)threadIdx.x, pieces); }
    __device__ __forceinline__ Piece load(int j) const {
        const int e = from(piece(j));
        Piece p;
        if (vocab >= V) {
            p.raw = *(const Loaded*)(row + e);
            if (MASK)
#pragma unroll
                for (int k = 0; k < V / 4; k++) p.bits[k] = *(const Bits*)(mask + e + 4 * k);
        } else
#pragma unroll
            for (int k = 0; k < V; k++) {
                p.raw[k] = row[min(k, vocab - 1)];
                if (MASK) p.bits[k / 4] = (k % 4 ? p.bits[k / 4] : 0) | (unsigned)(mask[min(k, vocab - 1)] != 0) << (k % 4 * 8);
            }
        return p;
    }
    // its logits; what is masked, what a moved piece has of others and what is behind the row is -inf
    __device__ __forceinline__ void logits(int j, const Piece& p, float (&y)[V]) const {
#pragma unroll
        for (int k = 0; k < V; k++) y[k] = (float)p.raw[k];
        if (j == 0 || j >= rounds - 1) {
            const int b = begin(piece(j)), e = from(piece(j));
#pragma unroll
            for (int k = 0; k < V; k++)
                if (e + k < b || e + k >= min(b + V, vocab)) y[k] = -INFINITY;
        }
        if (MASK) {
            unsigned any = p.bits[0];
#pragma unroll
            for (int k = 1; k < V / 4; k++) any |= p.bits[k];
            if (__ballot(any != 0))
#pragma unroll
                for (int k = 0; k < V; k++) y[k] = p.bits[k / 4] & 0xffu << (k % 4 * 8) ? -INFINITY : y[k];
        }
    }
    // f(piece, its logits), AHEAD pieces on their way
    template <int AHEAD, typename F>
    __device__ __forceinline__ void each_piece(F f) const {
        Piece p[AHEAD];
#pragma unroll
        for (int d = 0; d < AHEAD; d++) p[d] = load(d);
#pragma unroll 1
        for (int j0 = 0; j0 < rounds; j0 += AHEAD)
#pragma unroll
            for (int d = 0; d < AHEAD; d++) {
                const int j = j0 + d;
                if (j >= rounds) break;
                float y[V];
                const Piece now = p[d];
                p[d] = load(j + AHEAD);
                logits(j, now, y);
                f(j * THREADS + (int)threadIdx.x, y);
            }
    }
    // f(x, id) of the tokens, one at a time: little code, for what is hardly ever needed
    template <typename F>
    __device__ __forceinline__ void each_slowly(F f) const {
#pragma unroll 1
        for (int id = threadIdx.x; id < vocab; id += THREADS) {
            const float x = MASK && mask[id] ? -INFINITY : (float)row[id];
            if (x > -INFINITY) f(x, id);
        }
    }
    // f(x, id) of the tokens not below v
    template <int AHEAD, typename F>
    __device__ __forceinline__ void each_from(float v, F f) const {
        each_piece<AHEAD>([&](int p, const float (&y)[V]) {
            float most = y[0];
#pragma unroll
            for (int k = 1; k < V; k++) most = fmaxf(most, y[k]);
            if (!(most >= v)) return;
            const int e = from(min(p, pieces));
#pragma unroll
            for (int k = 0; k < V; k++)
                if (y[k] >= v && y[k] > -INFINITY) f(y[k], e + k);
        });
    }
};

struct Shared {
    u64 sums[BINS];
    u64 wave_sum[WAVES];
    u64 before, here;
    unsigned at, lo, hi;
    int n;
    float lx[LIST];
    int lid[LIST];
};

// sh.sums summed up: this thread's in `mine`, the sum up to and with it, and of all
__device__ __forceinline__ u64 running(Shared& sh, u64& mine, u64& all) {
    const int tid = threadIdx.x, wave = tid >> 6;
    mine = sh.sums[tid];
    const u64 run = wave_running(mine);
    if ((tid & 63) == 63) sh.wave_sum[wave] = run;
    __syncthreads();
    all = 0;
    u64 front = 0;
#pragma unroll
    for (int k = 0; k < WAVES; k++) {
        if (k == wave) front = all;
        all += sh.wave_sum[k];
    }
    return run + front;
}

template <typename T, bool MASK>
__global__ void __launch_bounds__(THREADS) sample_kernel(MzSample a, int shift) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63;
    const long r = blockIdx.x, n = a.at ? (long)*a.at + a.at_add : 0;
    if (n < 0 || n >= a.stride) return;
    const long at = r * a.stride + n;
    Row<T, MASK> row;
    row.open(a, r);
    const float t = a.temperatures ? a.temperatures[r] : a.temperature, top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    const float min_p = a.min_ps ? a.min_ps[r] : a.min_p, u0 = a.u[at];
    const int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    auto answer = [&](int token, float logp, int kept) {
        a.tokens[at] = token;
        if (a.logp) a.logp[at] = logp;
        if (a.kept) a.kept[at] = kept;
    };

    float best = -INFINITY;  // this thread's largest
    unsigned count = 0;      // tokens
    bool nan = false;
    row.template each_piece<4>([&](int, auto& y) {
#pragma unroll
        for (int k = 0; k < row.V; k++) {
            best = fmaxf(best, y[k]);
            count += y[k] > -INFINITY;
            nan |= y[k] != y[k];
        }
    });
    const float top = block_all(best, Max());
    count = block_all(count | (nan ? 1u << 31 : 0), [](unsigned x, unsigned y) { return ((x | y) & 1u << 31) | ((x + y) & 0x7fffffff); });
    const bool bad = count >> 31 || top == INFINITY || !(t >= 0.f) || t == INFINITY || top_p != top_p || min_p != min_p;
    if (bad || !count) {
        if (tid == 0) answer(-1, bad ? NAN : -INFINITY, 0);
        return;
    }
    if (t == 0.f || top_k == 1 || top_p <= 0.f) {  // the first
        unsigned id = ~0u;
        row.template each_from<4>(top, [&](float, int i) { id = min(id, (unsigned)i); });
        id = block_all(id, Min());
        if (tid == 0) answer((int)id, 0.f, 1);
        return;
    }
    const double per = 1.4426950408889634 / (double)t;
    const Weights weight = {(double)top, per, -200.0 / per, shift};
    const float u = u0 >= 0.f ? fminf(u0, 0x1.fffffep-1f) : 0.f;
    const bool limit_k = top_k > 0 && (unsigned)top_k < count, limit_p = top_p < 1.f, limit_m = min_p > 0.f;
    float low = -INFINITY;  // the lowest logit of weight min_p or more
    if (limit_m) {
        const double l = (double)top + (double)t * log(fmin((double)min_p, 1.0));
        low = (float)l;
        if ((double)low < l) low = value_at(order_of(low) - 1);
    }
    // intervals of values: 32 to a factor of two of weights, the last one without an end
    const float per_bin = 32.f * (float)per;
    auto value_bin = [&](float x) { return (int)fminf((top - x) * per_bin, BINS - 1.f); };

    // Limits so far: tokens of an order below cut's, or cut's with an id up to last.
    unsigned cut = ~0u;
    int last = 0;
    auto inside = [&](float x, int id) {
        const unsigned o = order_of(x);
        return o < cut || (o == cut && id <= last);
    };
    // the same, and not below `low`, with few instructions
    struct Edge {
        float least, tie;
        int last;
        __device__ __forceinline__ bool has(float x, int id) const { return x >= least && !(x == tie && id > last); }
    };
    auto edge_of = [&](float low) {
        return Edge{cut == ~0u ? low : fmaxf(low, value_at(cut)), cut == ~0u ? NAN : value_at(cut), last};
    };
    u64 total = 0;        // what top_p is a share of
    bool listed = false;  // all tokens that the limits can leave are in the list: this thread's
    int m = 0;            // its length
    float lx = -INFINITY;
    int lid = 0;
    // tokens not below `from` in intervals `first` to `final` into the list; whether it holds them all
    auto gather = [&](float from, int first, int final) {
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
        row.template each_from<4>(from, [&](float x, int id) {
            const int b = value_bin(x);
            if (b < first || b > final || !inside(x, id)) return;
            const int i = atomicAdd(&sh.n, 1);
            if (i < LIST) {
                sh.lx[i] = x;
                sh.lid[i] = id;
            }
        });
        __syncthreads();
        m = sh.n;
        lx = tid < m ? sh.lx[tid] : -INFINITY;
        lid = tid < m ? sh.lid[tid] : 0;
        return m <= LIST;
    };
    auto logp_of = [&](float x, u64 sum) { return (float)(((double)x - (double)top) / (double)t - log(ldexp((double)sum, -shift))); };

    // The lowest order, of values or of ids, for which the sum of weights (`unit`: of ones) over what `each` has of that order and
    // below, with `before` in front, is at least need (`above`: more); the sums in front of it and of it. Each pass sums up
    // intervals; of the one with the place the range is found and divided again.
    u64 before = 0, here = 0;
    int id_bits = 0;
    while ((a.vocab - 1) >> id_bits >= BINS) id_bits++;
    auto search = [&](const auto& each, bool by_id, bool unit, double need, bool above) {
        unsigned lo = 0, hi = ~0u;
        int bits = -1;  // (of the first pass: none)
        for (;;) {
            __syncthreads();
            sh.sums[tid] = 0;
            if (tid == 0) {
                sh.lo = ~0u;
                sh.hi = 0;
            }
            __syncthreads();
            auto order = [&](float x, int id) { return by_id ? (unsigned)id : order_of(x); };
            auto bin = [&](float x, int id) { return bits >= 0 ? (int)((order(x, id) - lo) >> bits) : by_id ? id >> id_bits : value_bin(x); };
            auto ranged = [&](float x, int id) { return order(x, id) >= lo && order(x, id) <= hi; };
            each([&](float x, int id) {
                if (ranged(x, id)) atomicAdd(&sh.sums[bin(x, id)], unit ? 1 : weight(x));
            });
            __syncthreads();
            u64 mine, all;
            const u64 run = running(sh, mine, all) + before;
            auto passes = [&](u64 s) { return above ? (double)s > need : (double)s >= need; };
            if (passes(run) && !passes(run - mine)) {  // one thread's
                sh.before = run - mine;
                sh.here = mine;
                sh.at = tid;
            }
            __syncthreads();
            before = sh.before;
            here = sh.here;
            const int place = (int)sh.at;
            if (bits == 0) return lo + place;
            unsigned l = ~0u, h = 0;
            each([&](float x, int id) {
                if (ranged(x, id) && bin(x, id) == place) {
                    l = min(l, order(x, id));
                    h = max(h, order(x, id));
                }
            });
            if (l <= h) {
                atomicMin(&sh.lo, l);
                atomicMax(&sh.hi, h);
            }
            __syncthreads();
            lo = sh.lo;
            hi = sh.hi;
            if (lo == hi) return lo;
            bits = max(0, 32 - __clz(hi - lo) - BIN_BITS);
        }
    };

    // top_k, then top_p (in a loop: the code is there once)
#pragma unroll 1
    for (int stage = limit_k ? 0 : 1; stage < (limit_p ? 2 : 1); stage++) {
        const bool unit = stage == 0;
        double need = unit ? (double)top_k : 0.0;
        bool ready = listed;  // the list has what is needed
        bool known = false;   // what can be needed is not below `from`
        float from = -INFINITY;
        int place = BINS - 1;
        before = 0;
        if (unit && top_k <= LIST / 2 && __syncthreads_count(best > -INFINITY) >= top_k) {
            // Not below the k-th of the threads' best logits, or the least of those in the intervals up to it.
            const int b = best > -INFINITY ? value_bin(best) : BINS - 1;
            __syncthreads();
            sh.sums[tid] = 0;
            __syncthreads();
            if (best > -INFINITY) atomicAdd(&sh.sums[b], 1);
            __syncthreads();
            u64 mine, all;
            const u64 run = running(sh, mine, all);
            if (run >= (u64)top_k && run - mine < (u64)top_k) sh.at = tid;
            __syncthreads();
            const float edge = block_all(b <= (int)sh.at ? best : INFINITY, Min());
            from = limit_p ? edge : fmaxf(edge, low);
            known = true;
        }
        // The list: first, not below `from`; then, with the intervals' sums, the tokens up to the end of the one that has the limit;
        // then that interval's.
        u64 front = 0;
        for (int attempt = known ? 0 : 1; !ready && attempt < 3; attempt++) {
            if (attempt == 1) {
                __syncthreads();
                sh.sums[tid] = 0;
                __syncthreads();
                u64 rest = 0;  // of the last interval
                const Edge edge = edge_of(-INFINITY);
                row.template each_piece<1>([&](int p, auto& y) {
                    const int e = row.from(min(p, row.pieces));
                    u64 w[row.V];
                    int b[row.V];
#pragma unroll
                    for (int k = 0; k < row.V; k++) {
                        w[k] = unit ? y[k] > -INFINITY : weight(y[k]);
                        if (!edge.has(y[k], e + k)) w[k] = 0;
                        b[k] = value_bin(y[k]);
                        if (b[k] == BINS - 1) rest += w[k];
                    }
#pragma unroll
                    for (int k = 0; k < row.V; k++)
                        if (b[k] < BINS - 1) atomicAdd(&sh.sums[b[k]], w[k]);
                });
                rest = block_all(rest, Add());
                if (tid == BINS - 1) sh.sums[tid] = rest;
                __syncthreads();
                u64 mine, all;
                const u64 run = running(sh, mine, all);
                if (!unit) {
                    total = all;
                    need = (double)top_p * (double)total;
                }
                if ((double)run >= need && !((double)(run - mine) >= need)) {
                    sh.before = run - mine;
                    sh.at = tid;
                }
                __syncthreads();
                place = (int)sh.at;
                front = sh.before;
                // (not above any of the interval's: a product more than exact ends of it)
                from = place == BINS - 1 ? -INFINITY : top - (place + 1.01f) * 1.00001f / per_bin;
                from = from > -INFINITY ? from : -INFINITY;
            }
            ready = gather(from, attempt == 2 ? place : 0, place);
            listed = ready && attempt < 2;
            if (ready && attempt == 2) before = front;
        }
        if (!unit && total == 0) {
            total = block_all(lx > -INFINITY && inside(lx, lid) ? weight(lx) : 0, Add());
            need = (double)top_p * (double)total;
        }
        if (listed && m <= 64) break;  // (one wave does it all)
        if (unit && listed && m < top_k) continue;  // (min_p has left fewer: no limit)
        bool ties = false, by_id = false, ones = unit;
        const unsigned was = cut;
        const int until = last;
#pragma unroll 1
        for (;;) {
            auto each = [&](auto f) {
                auto in = [&](float x, int id) { return ties ? order_of(x) == cut : inside(x, id); };
                if (ready) {
                    if (lx > -INFINITY && in(lx, lid)) f(lx, lid);
                } else
                    row.each_slowly([&](float x, int id) { if (in(x, id)) f(x, id); });
            };
            const unsigned o = search(each, by_id, ones, need, false);
            if (ties) {
                last = min((int)o, last);
                break;
            }
            const u64 every = unit ? 1 : weight(value_at(o));  // (of each token of that value)
            // as many of them as it takes, the lower ids first
            const double some0 = ceil((need - (double)before) / (double)every);
            u64 some = some0 > 1.0 ? (u64)some0 : 1;
            while (some > 1 && (double)(before + (some - 1) * every) >= need) some--;
            while ((double)(before + some * every) < need && some * every < here) some++;
            cut = o;
            last = o == was ? until : a.vocab;
            if (some * every >= here) break;
            ties = by_id = ones = true;
            need = (double)some;
            before = 0;
        }
    }
    if (!limit_k && !limit_p && limit_m) listed = gather(low, 0, BINS - 1);

    if (listed && m <= 64) {
        if (tid >= 64) return;
        const Key k = sorted_wave(lx > -INFINITY ? key_of(lx, lid) : 0, lane);
        const float x = value_of(k);
        const u64 w = k ? weight(x) : 0, run = wave_running(w);
        if (limit_k) total = lane_key(run, min(top_k, 64) - 1);
        const bool keep = k && !(limit_k && lane >= top_k) && !(limit_p && lane && (double)(run - w) >= (double)top_p * (double)total) && x >= low;
        const int c = __popcll(__ballot(keep));
        const u64 sum = lane_key(run, c - 1);
        const Key by_id = sorted_wave(keep ? (Key)(IDS - 1 - id_of(k)) << 32 | __builtin_bit_cast(unsigned, x) : 0, lane);
        const float y = __builtin_bit_cast(float, (unsigned)by_id);
        const u64 upto = wave_running(by_id ? weight(y) : 0);
        const int i = __ffsll((unsigned long long)__ballot((double)upto > (double)u * (double)sum)) - 1;
        if (lane == i) answer((int)(IDS - 1 - (unsigned)(by_id >> 32)), logp_of(y, sum), c);
        return;
    }

    auto kept = [&](float x, int id) { return x >= low && inside(x, id); };
    u64 sum = 0;
    unsigned c = 0, drawn;
    if (listed) {
        auto each = [&](auto f) {
            if (lx > -INFINITY && kept(lx, lid)) f(lx, lid);
        };
        each([&](float x, int) {
            sum += weight(x);
            c++;
        });
        sum = block_all(sum, Add());
        before = 0;
        drawn = search(each, true, false, (double)u * (double)sum, true);
    } else {
        // Sums of 16 pieces or more each, then the token among those that the sum with it has, by ids.
        int piece_bits = 4;
        while ((row.pieces - 1) >> piece_bits >= BINS) piece_bits++;
        __syncthreads();
        sh.sums[tid] = 0;
        __syncthreads();
        const Edge edge = edge_of(low);
        row.template each_piece<1>([&](int p, auto& y) {
            const int e = row.from(min(p, row.pieces));
            u64 w = 0;
#pragma unroll
            for (int k = 0; k < row.V; k++) {
                const u64 v = weight(y[k]);
                const bool in = edge.has(y[k], e + k);
                w += in ? v : 0;
                c += in && y[k] > -INFINITY;
            }
            w = row_all(w, Add());
            if ((tid & 15) == 0) atomicAdd(&sh.sums[p >> piece_bits], w);
        });
        __syncthreads();
        u64 mine;
        const u64 run = running(sh, mine, sum);
        const double need = (double)u * (double)sum;
        if ((double)run > need && !((double)(run - mine) > need)) {
            sh.before = run - mine;
            sh.at = tid;
        }
        __syncthreads();
        const int place = (int)sh.at;
        before = sh.before;
        // (with 16 pieces of 8 logits at most 128: a thread each)
        const int first = place << piece_bits, pieces = 1 << piece_bits;
        for (int p0 = 0; ; p0 += THREADS / row.V) {
            __syncthreads();
            sh.sums[tid] = 0;
            const int p = first + p0 + tid / row.V, id = row.begin(p) + tid % row.V;
            float x = -INFINITY;
            if (p0 + tid / row.V < pieces && id >= 0 && id < row.vocab && !(MASK && row.mask[id])) x = (float)row.row[id];
            sh.sums[tid] = edge.has(x, id) ? weight(x) : 0;
            __syncthreads();
            u64 mine, all;
            const u64 run = running(sh, mine, all) + before;
            if ((double)run > need && !((double)(run - mine) > need)) sh.n = id;
            before += all;
            if (__syncthreads_or((double)run > need) || p0 + THREADS / row.V >= pieces) break;
        }
        drawn = (unsigned)sh.n;
    }
    c = block_all(c, Add());
    if (tid == 0) answer((int)drawn, logp_of((float)row.row[drawn], sum), (int)c);
}

// weights are multiples of 2^-shift: a row's sum stays below 2^62, and a weight has at most 52 bits
int shift_of(int vocab) {
    int bits = 0;
    while ((1L << bits) < vocab) bits++;
    return std::min(51, 62 - bits);
}

template <typename T>
void launch(hipStream_t s, const MzSample& p) {
    const dim3 grid(p.rows), block(THREADS);
    if (p.mask) hipLaunchKernelGGL((sample_kernel<T, true>), grid, block, 0, s, p, shift_of(p.vocab));
    else hipLaunchKernelGGL((sample_kernel<T, false>), grid, block, 0, s, p, shift_of(p.vocab));
}

}  // namespace

size_t mz_sample_work(const MzSample& p) { return 0; }

hipError_t mz_sample_launch(hipStream_t s, const MzSample& p) {
    if (p.half) launch<f16>(s, p);
    else launch<float>(s, p);
    return hipGetLastError();
}
