// The next token of rows of logits (mz_sample_args in mimizuku.h).
//
// The kept tokens are the first ones in the order of falling logits, of equal ones the lower id first: those with a logit above
// some value, and of those with that value the ids up to some id. So each limit is a pair (value, id), the kept set is what
// passes the highest of them, and no row is sorted. Where a limit lies is found by sums over intervals of values, the one that
// holds it taken apart again.
//
// Weights are whole multiples of 2^-shift: sums of them are exact in 64 bits whatever their order.
//
// A workgroup of 1024 threads takes a row and reads it again for each pass, from the caches after the first; the largest logit of
// each 16-byte piece stays in LDS, so that passes for a few tokens skip the other pieces. Limits leave few tokens of most rows:
// those that the limits can reach go into a list, and up to 64 of them are put in order by one wave.
//
// What bounds it is the vector unit and the passes' latency, not memory: a row is 16 waves of a CU whatever the number of rows, a
// weight about 20 instructions in 64 bits, a pass 3 to 9 us. A call among 20 back to back, rows of 51,866 with a dozen likely tokens:
// 7.3 us at temperature 0 (8.6 for 160 rows); one row with every limit 17 (a pass for the largest, lists, two sorts); 32 rows with
// top_p 0.9 36 to 47 at temperature 0.6 (a pass that counts tokens in intervals, one that sums the weights around the place
// exactly, one that draws; what the data leave near the place decides on a second sum; 4 of 40 draws of the data 58 to 61), 63 at 1;
// 160 rows without limits 24 (the largest, the sums by pieces); 1024 fp16 rows with settings of their own 160 to 170 (one workgroup a CU:
// four rows one after the other, each idle at its barriers). Where many logits are equal or nearly so a place is looked for among
// the whole row's tokens: 32 such rows take 213 with top_p 0.9, with equal logits and top_k 400 230.
// Sums of weights by floating-point atomics in LDS were slower than counts and depend on the order; whole rows in registers need
// more of them than 16 waves leave.
#include <algorithm>

#include "mz_common.h"
#include "mz_keys.h"
#include "mz_kernels.h"

namespace {

typedef unsigned long long u64;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int BINS = THREADS, BIN_BITS = 10, LIST = THREADS;
constexpr int MOST_ROUNDS = 30;  // pieces of a thread that have a word of LDS

// a logit as a number in the opposite order, -0 and +0 alike
__device__ __forceinline__ unsigned order_of(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v + 0.f);
    return u ^ (~(unsigned)((int)u >> 31) & 0x7fffffffu);
}
__device__ __forceinline__ float value_at(unsigned o) { return __builtin_bit_cast(float, o ^ (~(unsigned)((int)o >> 31) & 0x7fffffffu)); }

constexpr float LOWEST = -3.40282347e38f;

// exp((x - top) / t) in steps of 2^-shift of finite x. With s = (x - top) / (t ln 2), n the whole number next to it and f = s - n:
// n + shift is in the low bits of s + (1.5 * 2^52 + shift), 2^f is a polynomial of degree 8 through its values at nine Chebyshev
// nodes (relative error below 1.1e-12), n goes into its exponent, and the sum with 2^52 has the result, rounded, in its low 52 bits.
// What is 200 powers of two below the top has weight 0, as has what is next to the top where t is too small for it to count.
struct Weights {
    double top, per, magic;
    float lowest, inf;  // (inf: the median with a number that the compiler does not know is the larger one, in one instruction)
    double c[8];  // (in registers: as immediate numbers each would take two more instructions)
    __device__ __forceinline__ Weights(float top_, float t, int shift) {
        const double gap = (double)top_ - (double)fmaxf(value_at(order_of(top_) + 1), LOWEST);  // to the next number below
        top = top_;
        per = 1.4426950408889634 / (double)t;
        double far = (double)t * (200.0 / 1.4426950408889634);
        if (far < gap) {
            per = 200.0 / gap;
            far = gap;
        }
        magic = 0x1.8p52 + shift;
        lowest = fmaxf((float)(top - far), LOWEST);
        c[0] = 0x1.63d136366db24p-20;
        c[1] = 0x1.00dc4a532fb8ep-16;
        c[2] = 0x1.4308ac85aa947p-13;
        c[3] = 0x1.5d8745a728441p-10;
        c[4] = 0x1.3b2ab7181b755p-7;
        c[5] = 0x1.c6b08dd6fd234p-5;
        c[6] = 0x1.ebfbdff823cedp-3;
        c[7] = 0x1.62e42fef84cf0p-1;
#pragma unroll
        for (int i = 0; i < 8; i++) asm("" : "+v"(c[i]));
        inf = INFINITY;
        asm("" : "+s"(inf));
    }
    // of N logits side by side: each is a chain of dependent steps. RAW: with the bits above, ABOVE, for sums of whole pieces
    template <int N, bool RAW>
    __device__ __forceinline__ void of(const float* x, u64* to) const {
        double d[N], s[N], f[N], p[N];
#pragma unroll
        for (int k = 0; k < N; k++) d[k] = (double)__builtin_amdgcn_fmed3f(x[k], lowest, inf) - top;
#pragma unroll
        for (int k = 0; k < N; k++) s[k] = fma(d[k], per, magic);
#pragma unroll
        for (int k = 0; k < N; k++) f[k] = fma(d[k], per, magic - s[k]);
#pragma unroll
        for (int k = 0; k < N; k++) p[k] = fma(c[0], f[k], c[1]);
#pragma unroll
        for (int i = 2; i < 8; i++)
#pragma unroll
            for (int k = 0; k < N; k++) p[k] = fma(p[k], f[k], c[i]);
#pragma unroll
        for (int k = 0; k < N; k++) {
            u32x2 b = __builtin_bit_cast(u32x2, fma(p[k], f[k], 1.0));
            b[1] += __builtin_bit_cast(u32x2, s[k])[0] << 20;
            b = __builtin_bit_cast(u32x2, __builtin_bit_cast(double, b) + 0x1p52);
            if (!RAW) b[1] &= 0xfffffu;
            to[k] = __builtin_bit_cast(u64, b);
        }
    }
    __device__ __forceinline__ u64 operator()(float x) const {
        u64 w;
        of<1, false>(&x, &w);
        return w;
    }
    template <int V>
    __device__ __forceinline__ void of_piece(const float (&x)[V], u64 (&w)[V]) const {
#pragma unroll
        for (int k = 0; k < V; k += 4) of<4, false>(x + k, w + k);
    }
    // the sum of a piece's weights, of -inf too (`plain`)
    template <int V>
    __device__ __forceinline__ u64 sum_of_piece(const float (&x)[V]) const {
        u64 w[V], sum = 0;
#pragma unroll
        for (int k = 0; k < V; k += 4) of<4, true>(x + k, w + k);
#pragma unroll
        for (int k = 0; k < V; k++) sum += w[k];
        return sum - V * ABOVE;
    }
    static constexpr u64 ABOVE = 0x433ULL << 52;
    // whether -inf, taken as `lowest`, has weight 0: not where a temperature leaves every finite number a weight
    __device__ __forceinline__ bool plain() const { return lowest > LOWEST; }
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
    // (every lane reads another: there is no old value)
    if constexpr (sizeof(T) == 8) {
        const u32x2 b = __builtin_bit_cast(u32x2, v);
        return __builtin_bit_cast(T, u32x2{(unsigned)__builtin_amdgcn_mov_dpp((int)b[0], CTRL, 0xF, 0xF, true),
                                           (unsigned)__builtin_amdgcn_mov_dpp((int)b[1], CTRL, 0xF, 0xF, true)});
    } else
        return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
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
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved_in(u64 v) {
    const u32x2 b = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(u64, u32x2{(unsigned)__builtin_amdgcn_update_dpp(0, (int)b[0], CTRL, ROWS, 0xF, true),
                                         (unsigned)__builtin_amdgcn_update_dpp(0, (int)b[1], CTRL, ROWS, 0xF, true)});
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved_in(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, true));
}
template <typename T>
__device__ __forceinline__ T wave_running(T v) {
    v += moved_in<0x111, 0xF>(v);
    v += moved_in<0x112, 0xF>(v);
    v += moved_in<0x114, 0xF>(v);
    v += moved_in<0x118, 0xF>(v);
    v += moved_in<0x142, 0xA>(v);
    return v + moved_in<0x143, 0xC>(v);
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
    float* largest;          // of each piece, in LDS (null: some rows of the launch have too many)

    // lds: null, or a word for each piece that a row of this length can have wherever it begins (see launch: which of the two is
    // decided there, for all rows alike)
    __device__ __forceinline__ void open(const MzSample& a, long r, float* lds) {
        row = (const T*)a.logits + r * a.ld;
        mask = a.mask;
        vocab = a.vocab;
        off = (int)((uintptr_t)row % 16 / sizeof(T));
        pieces = (vocab + off + V - 1) / V;
        rounds = (pieces + THREADS - 1) / THREADS;
        largest = lds ? lds + threadIdx.x : nullptr;
    }
    // where this thread's piece j begins, and where it is read: pieces at the row's ends are moved into it
    __device__ __forceinline__ int begin(int j) const { return (j * THREADS + (int)threadIdx.x) * V - off; }
    __device__ __forceinline__ int from(int j) const {
        const int e = begin(j);
        return j == 0 || j >= rounds - 1 ? max(min(e, vocab - V), 0) : e;
    }
    __device__ __forceinline__ Piece load(int j) const {
        const int e = from(j);
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
            const int b = begin(j), e = from(j);
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
    // f(j, its logits), AHEAD pieces on their way
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
                f(j, y);
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
    // f(x, id) of the tokens not below v; pieces whose largest is are not read
    template <typename F>
    __device__ __forceinline__ void each_from(float v, F f) const {
        unsigned has = 0;  // this thread's pieces
        if (largest)
#pragma unroll 4
            for (int j = 0; j < rounds; j++) has |= (unsigned)(largest[j * THREADS] >= v) << j;
        int j = -1;
        auto next = [&]() {
            if (!largest) return j + 1;
            const int i = has ? __ffs(has) - 1 : rounds;
            has &= has - 1;
            return i;
        };
        j = next();
        if (j >= rounds) return;
        Piece p = load(j);
        do {
            const Piece now = p;
            const int at = j;
            j = next();
            if (j < rounds) p = load(j);  // on its way while this one is taken
            float y[V];
            logits(at, now, y);
            const int e = from(at);
#pragma unroll
            for (int k = 0; k < V; k++)
                if (y[k] >= v && y[k] > -INFINITY) f(y[k], e + k);
        } while (j < rounds);
    }
};

struct Shared {
    u64 sums[BINS];
    float wave_about[WAVES], about;
    float wave_best[WAVES];
    unsigned wave_count[WAVES];
    u64 wave_sum[WAVES];
    u64 before, here;
    unsigned at, drawn_x;
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
__global__ void __launch_bounds__(THREADS) sample_kernel(MzSample a, int shift, int words) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63;
    const long r = blockIdx.x, n = a.at ? (long)*a.at + a.at_add : 0;
    if (n < 0 || n >= a.stride) return;
    const long at = r * a.stride + n;
    extern __shared__ float largest[];
    Row<T, MASK> row;
    row.open(a, r, words ? largest : nullptr);
    const float t = a.temperatures ? a.temperatures[r] : a.temperature, top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    const float min_p = a.min_ps ? a.min_ps[r] : a.min_p, u0 = a.u[at];
    const int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    auto answer = [&](int token, float logp, int kept) {
        a.tokens[at] = token;
        if (a.logp) a.logp[at] = logp;
        if (a.kept) a.kept[at] = kept;
    };

    float inf = INFINITY;  // (the median with a number that the compiler does not know is the larger one, in one instruction)
    asm("" : "+s"(inf));
    float best = -INFINITY;  // this thread's largest
    unsigned count = 0;      // tokens
    bool nan = false;
    row.template each_piece<4>([&](int j, auto& y) {
        float most = y[0];
#pragma unroll
        for (int k = 1; k < row.V; k++) most = __builtin_amdgcn_fmed3f(most, y[k], inf);
#pragma unroll
        for (int k = 0; k < row.V; k++) {
            count += y[k] > -INFINITY;
            nan |= y[k] != y[k];
        }
        best = __builtin_amdgcn_fmed3f(best, most, inf);
        if (row.largest) row.largest[j * THREADS] = most;
    });
    {
        const float m = wave_max(best);
        unsigned c = row_all(count, Add());
        c = lane_of(c, 0) + lane_of(c, 16) + lane_of(c, 32) + lane_of(c, 48);
        const bool any = __ballot(nan);
        if (lane == 0) {
            sh.wave_best[tid >> 6] = m;
            sh.wave_count[tid >> 6] = any ? 1u << 31 : c;
        }
    }
    __syncthreads();
    const float top = row_all(sh.wave_best[lane & 15], Max());
    count = row_all(sh.wave_count[lane & 15], [](unsigned x, unsigned y) { return (x | y) >> 31 ? 1u << 31 : x + y; });
    const bool bad = count >> 31 || top == INFINITY || !(t >= 0.f) || t == INFINITY || top_p != top_p || min_p != min_p;
    if (bad || !count) {
        if (tid == 0) answer(-1, bad ? NAN : -INFINITY, 0);
        return;
    }
    if (t == 0.f || top_k == 1 || top_p <= 0.f || min_p > 1.f) {  // the first
        unsigned id = ~0u;
        row.each_from(top, [&](float, int i) { id = min(id, (unsigned)i); });
        id = block_all(id, Min());
        if (tid == 0) answer((int)id, 0.f, 1);
        return;
    }
    const Weights weight(top, t, shift);
    const float u = u0 >= 0.f ? fminf(u0, 0x1.fffffep-1f) : 0.f;
    const bool limit_k = top_k > 0 && (unsigned)top_k < count, limit_p = top_p < 1.f, limit_m = min_p > 0.f;
    float low = -INFINITY;  // the lowest logit of weight min_p or more
    if (limit_m) {
        const double l = (double)top + (double)t * log((double)min_p);
        low = (float)l;
        if ((double)low < l) low = value_at(order_of(low) - 1);
    }
    // intervals of values, the last one without an end
    float per_bin = 1.f;
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
        __device__ __forceinline__ bool has(float x, int id) const { return (x >= least) & ((x != tie) | (id <= last)); }
    };
    auto edge_of = [&](float low) {
        return Edge{fmaxf(cut == ~0u ? low : fmaxf(low, value_at(cut)), LOWEST), cut == ~0u ? NAN : value_at(cut), last};
    };
    u64 total = 0;        // what top_p is a share of
    bool listed = false;  // all tokens that the limits can leave are in the list: this thread's
    int m = 0;            // its length
    float lx = -INFINITY;
    int lid = 0;
    // tokens from `from` to `upto` into the list; whether it holds them all
    auto gather = [&](float from, float upto) {
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
        row.each_from(from, [&](float x, int id) {
            if (x > upto || !inside(x, id)) return;
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
    // below, with `before` in front, is at least need (`above`: more); the sums in front of it and of it. The range of what is
    // left is divided into intervals, until one with the place is a single order.
    u64 before = 0, here = 0;
    auto search = [&](const auto& each, bool by_id, bool unit, double need, bool above) {
        auto order = [&](float x, int id) { return by_id ? (unsigned)id : order_of(x); };
        unsigned lo = 0, hi = ~0u;
        for (;;) {
            unsigned l = ~0u, h = 0;
            each([&](float x, int id) {
                const unsigned o = order(x, id);
                if (o >= lo && o <= hi) {
                    l = min(l, o);
                    h = max(h, o);
                }
            });
            lo = block_all(l, Min());
            hi = block_all(h, Max());
            sh.sums[tid] = 0;
            __syncthreads();
            const int bits = max(0, 32 - __clz(hi - lo) - BIN_BITS);
            each([&](float x, int id) {
                const unsigned o = order(x, id);
                if (o >= lo && o <= hi) atomicAdd(&sh.sums[(o - lo) >> bits], unit ? 1 : weight(x));
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
            lo += sh.at << bits;
            if (bits == 0) return lo;
            hi = min(hi, lo + (1u << bits) - 1);
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
        before = 0;
        if (unit) {  // down to the least of the threads' best logits, or of all
            const bool few = __syncthreads_count(best > -INFINITY) >= top_k;
            float least = few && best > -INFINITY ? best : top;
            if (!few)
                row.template each_piece<2>([&](int j, auto& y) {
#pragma unroll
                    for (int k = 0; k < row.V; k++) least = y[k] > -INFINITY ? fminf(least, y[k]) : least;
                });
            least = block_all(least, Min());
            per_bin = least < top ? BINS * 0.9999f / (top - least) : 1.f;
            known = few && top_k <= LIST / 2;
        } else  // 32 to a factor of two of weights
            per_bin = 32.f * (float)weight.per;
        if (known) {
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
        }
        if (known) ready = listed = gather(from, INFINITY);
        if (!ready) {
            // About where: the tokens of each interval, counted, with its middle's weight.
            __syncthreads();
            sh.sums[tid] = 0;
            __syncthreads();
            unsigned* const counts = (unsigned*)sh.sums;
            const Edge edge = edge_of(-INFINITY);
            const bool uncut = cut == ~0u;
            // (what is in none goes to a word of the thread's own: a branch around each atomic takes longer)
            auto count_in = [&](auto in) {
                row.template each_piece<2>([&](int j, auto& y) {
                    const int e = row.from(j);
#pragma unroll
                    for (int k = 0; k < row.V; k++) {
                        const unsigned b = (unsigned)((top - y[k]) * per_bin);  // (infinity: the largest number)
                        atomicAdd(&counts[(b < BINS - 1) & in(y[k], e + k) ? b : BINS + tid], 1);
                    }
                });
            };
            if (uncut) count_in([](float, int) { return true; });
            else count_in([&](float x, int id) { return edge.has(x, id); });
            __syncthreads();
            // (the last one has the others)
            const unsigned rest = (uncut ? count : (unsigned)top_k) - block_all(tid < BINS - 1 ? counts[tid] : 0, Add());
            const unsigned here_n = tid == BINS - 1 ? rest : counts[tid];
            const float w = unit ? 1.f : __builtin_amdgcn_exp2f((tid + 0.5f) * (-1.f / 32.f));
            __syncthreads();
            sh.sums[tid] = here_n;
            const float sum = wave_running(here_n * w);
            if (lane == 63) sh.wave_about[tid >> 6] = sum;
            __syncthreads();
            float every = 0.f, ahead = 0.f;
#pragma unroll
            for (int k = 0; k < WAVES; k++) {
                if (k == tid >> 6) ahead = every;
                every += sh.wave_about[k];
            }
            const float about = ahead + sum;
            u64 mine, all;
            const u64 run = running(sh, mine, all);
            float goal = unit ? (float)top_k : top_p * every, off = 0.f;
            // (the next attempt knows what a sum really is)
            for (int attempt = 0; attempt < 4; attempt++) {
                const int first = block_all(about + off >= goal ? tid : BINS - 1, Min());
                // With what is in front of it, and some behind, if that is few enough for one wave; otherwise some intervals around it:
                // 256 tokens on either side (with 128 the place is missed more often, which takes 32 rows from 45 us to 58: 9 times of
                // 40 at temperature 0.6 and top_p 0.9, 4 with 256; 8 and 3 of 10 at 1 and 0.5).
                if (tid == first) {
                    sh.before = run - mine;
                    sh.here = run;
                }
                __syncthreads();
                const bool few = sh.here <= 56;
                const u64 room = few ? 0 : 256;
                const int b0 = few ? 0 : block_all(run - mine + room >= sh.before ? tid : BINS - 1, Min());
                const int b1 = block_all(run <= (few ? 60 : sh.here + room) ? tid : 0, Max());
                const int end = max(b1, first) + 1;
                const float high = b0 ? top - b0 / per_bin : INFINITY;
                from = end >= BINS ? LOWEST : fmaxf(top - end / per_bin, LOWEST);
                if (tid == b0) sh.about = about - here_n * w;
                // Exactly: what is in front of these, and all.
                u64 in_front = 0, sums = 0;
                if (unit)
                    row.template each_piece<1>([&](int j, auto& y) {
                        const int e = row.from(j);
#pragma unroll
                        for (int k = 0; k < row.V; k++) in_front += y[k] > high && edge.has(y[k], e + k);
                    });
                else if (!b0 && uncut && weight.plain())
                    row.template each_piece<1>([&](int, auto& y) { sums += weight.sum_of_piece(y); });
                else if (uncut && weight.plain())
                    row.template each_piece<1>([&](int, auto& y) {
                        u64 w[row.V];
                        weight.of_piece(y, w);
#pragma unroll
                        for (int k = 0; k < row.V; k++) {
                            sums += w[k];
                            in_front += y[k] > high ? w[k] : 0;
                        }
                    });
                else
                    row.template each_piece<1>([&](int j, auto& y) {
                        const int e = row.from(j);
                        u64 w[row.V];
                        weight.of_piece(y, w);
#pragma unroll
                        for (int k = 0; k < row.V; k++) {
                            w[k] = edge.has(y[k], e + k) ? w[k] : 0;
                            sums += w[k];
                            in_front += y[k] > high ? w[k] : 0;
                        }
                    });
                in_front = block_all(in_front, Add());
                if (!unit) {
                    total = block_all(sums, Add());
                    need = (double)top_p * (double)total;
                }
                if (!gather(from, high)) break;
                const u64 within = block_all(lx > -INFINITY ? unit ? 1 : weight(lx) : 0, Add());
                ready = (!b0 || (double)in_front < need) && (double)(in_front + within) >= need;
                listed = ready && !b0;
                before = ready ? in_front : 0;
                if (ready) break;
                const double scale = unit ? 1.0 : ldexp(1.0, -shift);
                goal = (float)(need * scale);
                off = (float)((double)in_front * scale) - sh.about;
                __syncthreads();
            }
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
    if (!limit_k && !limit_p && limit_m) listed = gather(low, INFINITY);

    if (listed && m <= 64) {
        if (tid >= 64) return;
        const Key k = sorted_wave(lx > -INFINITY ? key_of(lx, lid) : 0, lane);
        const float x = value_of(k);
        const u64 w = k ? weight(x) : 0, run = wave_running(w);
        if (limit_k && !total) total = lane_key(run, min(top_k, 64) - 1);
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
    float drawn_x;
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
        drawn_x = (float)row.row[drawn];
    } else {
        // Sums of 16 pieces or more each, then the token among those that the sum with it has, by ids.
        int piece_bits = 4;
        while ((row.pieces - 1) >> piece_bits >= BINS) piece_bits++;
        __syncthreads();
        sh.sums[tid] = 0;
        __syncthreads();
        const Edge edge = edge_of(low);
        const bool every = cut == ~0u && low == -INFINITY && weight.plain();
        if (every) {
            row.template each_piece<1>([&](int j, auto& y) {
                const u64 w = row_all(weight.sum_of_piece(y), Add());
                if ((tid & 15) == 0) atomicAdd(&sh.sums[(j * THREADS + tid) >> piece_bits], w);
            });
            c = tid == 0 ? count : 0;
        } else {
            auto sum_up = [&](auto in) {
                row.template each_piece<1>([&](int j, auto& y) {
                    const int e = row.from(j);
                    u64 each[row.V], w = 0;
                    weight.of_piece(y, each);
#pragma unroll
                    for (int k = 0; k < row.V; k++) {
                        const bool has = in(y[k], e + k);
                        w += has ? each[k] : 0;
                        c += has;
                    }
                    w = row_all(w, Add());
                    if ((tid & 15) == 0) atomicAdd(&sh.sums[(j * THREADS + tid) >> piece_bits], w);
                });
            };
            if (edge.last >= a.vocab || cut == ~0u) sum_up([&](float x, int) { return x >= edge.least; });
            else sum_up([&](float x, int id) { return edge.has(x, id); });
        }
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
            const int id = (first + p0 + tid / row.V) * row.V - row.off + tid % row.V;
            float x = -INFINITY;
            if (p0 + tid / row.V < pieces && id >= 0 && id < row.vocab && !(MASK && row.mask[id])) x = (float)row.row[id];
            sh.sums[tid] = edge.has(x, id) ? weight(x) : 0;
            __syncthreads();
            u64 mine, all;
            const u64 run = running(sh, mine, all) + before;
            if ((double)run > need && !((double)(run - mine) > need)) {
                sh.n = id;
                sh.drawn_x = __builtin_bit_cast(unsigned, x);
            }
            before += all;
            if (__syncthreads_or((double)run > need) || p0 + THREADS / row.V >= pieces) break;
        }
        drawn = (unsigned)sh.n;
        drawn_x = __builtin_bit_cast(float, sh.drawn_x);
    }
    c = block_all(c, Add());
    if (tid == 0) answer((int)drawn, logp_of(drawn_x, sum), (int)c);
}

// weights are multiples of 2^-shift: a row's sum stays below 2^62, and a weight has at most 52 bits
int shift_of(int vocab) {
    int bits = 0;
    while ((1L << bits) < vocab) bits++;
    return std::min(51, 62 - bits);
}

template <typename T>
void launch(hipStream_t s, const MzSample& p) {
    constexpr int V = 16 / sizeof(T);
    const dim3 grid(p.rows), block(THREADS);
    // of the row that has the most pieces, one that begins V - 1 elements behind a multiple of 16 bytes
    const long rounds = (((long)p.vocab + 2 * V - 2) / V + THREADS - 1) / THREADS;
    const int words = rounds <= MOST_ROUNDS ? (int)rounds * THREADS : 0;
    if (p.mask) hipLaunchKernelGGL((sample_kernel<T, true>), grid, block, words * 4, s, p, shift_of(p.vocab), words);
    else hipLaunchKernelGGL((sample_kernel<T, false>), grid, block, words * 4, s, p, shift_of(p.vocab), words);
}

}  // namespace

hipError_t mz_sample_launch(hipStream_t s, const MzSample& p) {
    if (p.half) launch<f16>(s, p);
    else launch<float>(s, p);
    return hipGetLastError();
}
