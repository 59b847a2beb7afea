// Token scores (mz_score_args in mimizuku.h): log probability of a given token, entropy and best alternatives of rows of
// logits, in one pass over them.
//
// With m a row's maximum, at element i0, S the sum of exp(x - m) over the others and U that of exp(x - m)(x - m):
// ln sum exp x = m + log1p(S), log p = (x - m) - log1p(S), entropy = log1p(S) - U / (1 + S). The last two terms are both
// positive and S does not hold the 1 of the maximum, so that sure rows (S far below 1) keep their digits.
//
// Many rows are bound by memory: 7,040 rows of 51,866 fp32 logits (1.46 GB) 220 us, 6.65 TB/s, which is why a wave works on
// 1024 elements while the next are on their way and looks for alternatives only where a chunk's best passes the list. One row
// is a chain of dependent steps, 8.1 us: launch and logits 3.5, joining its 13 workgroups 1.9, five alternatives 3 (the lists of
// the waves, and of the parts); 32 rows 10.5.
#include <algorithm>

#include "mz_common.h"
#include "mz_kernels.h"

namespace {

constexpr int PER_LANE = 16, CHUNK = 64 * PER_LANE;  // elements that a lane / a wave holds at a time
constexpr int PARTS = 64;                            // most waves that share a row: one lane each where they are joined
// Lanes whose best elements go into the list one after the other, more through the network (3,000 rows of 51,866 fp16 logits, 5
// / 16 alternatives: never more than one 84 / 116 us, up to three 78 / 107, eight 78 / 103, 16 78 / 104)
constexpr int FEW = 8;
constexpr float LOG2E = 1.4426950408889634f;

// What one wave knows of its elements: m, s, u, then its alternatives' keys, best first.
constexpr int HEAD = 4, MOST = HEAD + 2 * MZ_SCORE_ALTS;

// d = x - m to exp(d) and exp(d) d, 0 and 0 for -inf
__device__ __forceinline__ void add(float x, float m, float& s, float& u) {
    const float d = x - m, e = __builtin_amdgcn_exp2f(d * LOG2E);
    s += e;
    u = fmaf(e, fmaxf(d, -200.f), u);
}

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
// the best 16 of two sorted rows: the better of every pair of opposite places, put in order
__device__ __forceinline__ Key joined(Key a, Key b, int lane) {
    return cleaned(larger(a, moved<0x140>(b)), lane);
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
// the best 16 of the four rows' sorted ones, best first, in every row
__device__ __forceinline__ Key best_of_rows(Key k, int lane) {
    k = joined(k, other_row(k, lane), lane);
    return joined(k, other_half(k, lane), lane);
}
// the best 16 of the wave's 64 keys, best first, in every row
__device__ __forceinline__ Key best16(Key k, int lane) {
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
    return best_of_rows(k, lane);
}
// the best 16 of n <= 16 parts' lists, a row of lanes each
__device__ __forceinline__ Key best_of_parts(const float* part, int n, int alts, int lane) {
    const int words = HEAD + 2 * alts, k = lane & 15;
    Key r[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = 4 * j + (lane >> 4);
        r[j] = i < n && k < alts ? *(const Key*)(part + i * words + HEAD + 2 * k) : 0;
    }
    if (n > 4) r[0] = joined(r[0], r[1], lane);
    if (n > 8) r[0] = joined(r[0], joined(r[2], r[3], lane), lane);
    return best_of_rows(r[0], lane);
}
// the lane with the largest of the wave's keys (v: their values), at least one of them not 0
__device__ __forceinline__ int best_lane(float v, Key k) {
    unsigned long long has = __ballot(v == wave_max(v));
    int lane = __ffsll(has) - 1;
    for (has &= has - 1; has; has &= has - 1) {  // (hardly ever)
        const int other = __ffsll(has) - 1;
        if (lane_key(k, other) > lane_key(k, lane)) lane = other;
    }
    return lane;
}

// The row's results from its parts (words as above, one lane each) and its alternatives (lane k of a row of lanes: k). tok, xt:
// the given token and its logit.
__device__ __forceinline__ void finish(const MzScores& p, long o, const float* part, int parts, int lane, int tok, float xt, Key list) {
    const bool on = lane < parts;
    const float* mine = part + (on ? lane * (HEAD + 2 * p.alts) : 0);
    const float mi = on ? mine[0] : -INFINITY, si = on ? mine[1] : 0.f, ui = on ? mine[2] : 0.f;
    const float m = wave_max(mi);
    // one of the parts with the row's maximum holds the element that S leaves out; the others' maxima count in it
    const bool owner = lane == __ffsll((unsigned long long)__ballot(mi == m)) - 1;
    const float d = mi - m, e = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(d * LOG2E);
    const float t = si + 1.f;
    // (a part of NaN only has m -inf and s NaN)
    const float S = wave_sum(owner || si != si ? si : t * e), U = wave_sum(owner ? ui : e == 0.f ? 0.f : e * fmaf(t, d, ui));
    const bool bad = S != S || m == INFINITY;
    const float z = log1pf(S);
    if (lane == 0 && p.logp)
        p.logp[o] = tok < 0 ? 0.f : bad || tok >= p.vocab ? NAN : m == -INFINITY || xt == -INFINITY ? -INFINITY : (xt - m) - z;
    if (lane == 0 && p.entropy) p.entropy[o] = bad ? NAN : m == -INFINITY ? 0.f : z - U / (1.f + S);
    if (lane >= p.alts) return;
    if (p.alt_ids) p.alt_ids[o * p.alts + lane] = bad || !list ? -1 : id_of(list);
    if (p.alt_logp) p.alt_logp[o * p.alts + lane] = bad ? NAN : list ? (value_of(list) - m) - z : -INFINITY;
}

// A workgroup's share of a row, four waves taking chunks of 1024 elements in turn. Where `splits` workgroups share a row the
// last of them to end has the parts of all.
template <typename T, bool MASK>
__global__ void __launch_bounds__(256) score_kernel(MzScores p, int splits) {
    constexpr int V = 16 / sizeof(T), G = PER_LANE / V;  // elements of a 16-byte load, loads of a chunk
    typedef T TV __attribute__((ext_vector_type(V)));
    __shared__ __attribute__((aligned(8))) float lds[PARTS * MOST];
    __shared__ Key lists[64];  // of the waves' shares of the parts
    __shared__ Key bound;  // no element with a smaller key is an alternative of the row
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = blockIdx.x / splits, split = blockIdx.x - r * splits;
    const T* row = (const T*)p.logits + r * p.ld;
    const long n = p.at ? (long)*p.at + p.at_add : 0;
    if (n < 0 || n >= p.out_stride) return;
    if (tid == 0) bound = 0;
    __syncthreads();
    // the row's 16-byte pieces, the first of which begins `off` elements before it
    const int off = (int)((uintptr_t)row % 16 / sizeof(T));
    const int chunks = (p.vocab + off + CHUNK - 1) / CHUNK, share = (chunks + splits - 1) / splits;
    const int c0 = split * share, c1 = min(c0 + share, chunks);

    // Lane's element 0 of load j, a piece's first; the loads at the row's ends are moved into the row (`from`: where they
    // are then), and what they have of other pieces is left out.
    auto piece = [&](int c, int j) { return (c * G + j) * 64 * V + lane * V - off; };
    auto from = [&](int e) { return max(min(e, p.vocab - V), 0); };

    float m = -INFINITY, S = 0.f, U = 0.f;  // m of the wave, the sums of the lane
    bool first = true;        // nothing is in the list
    Key list = 0, least = 0;  // lane k of each row: alternative k; the last one, or a larger bound that another wave found
    // the given token and its logit, which each wait for a load
    const int tok = p.logp && n < p.token_stride ? p.tokens[r * p.token_stride + n] : -1;
    const bool known = tok >= 0 && tok < p.vocab;
    const float xt = (float)row[known ? tok : 0];
    const bool left_out = MASK && p.mask[known ? tok : 0];
    typedef TV __attribute__((aligned(sizeof(T)))) Piece;
    typedef unsigned Bits __attribute__((aligned(1)));
    TV raw[G];
    unsigned masks[PER_LANE / 4];
    auto fetch = [&](int c) {
#pragma unroll
        for (int j = 0; j < G; j++) {
            const int e = from(piece(c, j));
            raw[j] = __builtin_nontemporal_load((const Piece*)(row + e));
            if (MASK)
#pragma unroll
                for (int k = 0; k < V / 4; k++) masks[j * V / 4 + k] = *(const Bits*)(p.mask + e + 4 * k);
        }
    };
    int c = c0 + wave;
    if (p.vocab < V) {  // a row shorter than a piece: lane 0's
#pragma unroll
        for (int j = 0; j < PER_LANE; j++) {
            raw[j / V][j % V] = row[min(j, p.vocab - 1)];
            if (MASK) {
                const unsigned bit = (p.mask[min(j, p.vocab - 1)] != 0) << (j % 4 * 8);
                masks[j / 4] = j % 4 ? masks[j / 4] | bit : bit;
            }
        }
    } else if (c < c1) fetch(c);
    for (; c < c1; c += 4) {
        float x[PER_LANE];
#pragma unroll
        for (int j = 0; j < PER_LANE; j++) {
            x[j] = (float)raw[j / V][j % V];
            if (MASK) x[j] = masks[j / 4] & 0xffu << (j % 4 * 8) ? -INFINITY : x[j];
        }
        if (c + 4 < c1) fetch(c + 4);  // on its way while this one is taken
        if (c == 0 || c == chunks - 1)
#pragma unroll
            for (int j = 0; j < G; j++) {
                const int e = piece(c, j), at = from(e);
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const bool in = at + k >= e && at + k < min(e + V, p.vocab);
                    x[j * V + k] = in ? x[j * V + k] : -INFINITY;
                }
            }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < PER_LANE; j++) top = fmaxf(top, x[j]);
        int at;  // the lane's best element, the first one of equal ones
        auto find = [&]() {
            at = 0;
#pragma unroll
            for (int j = PER_LANE - 1; j >= 0; j--) at = x[j] == top ? j : at;
        };
        if (__ballot(top > m)) {  // a new maximum: the sums so far, the old maximum among them, become multiples of it
            find();
            const float mn = wave_max(top);
            const bool own = lane == __ffsll((unsigned long long)__ballot(top == mn)) - 1;
            if (m > -INFINITY) {
                const float d = m - mn, f = __builtin_amdgcn_exp2f(d * LOG2E);
                const float t = S + (lane == 0 ? 1.f : 0.f);
                U = f == 0.f ? 0.f * U : f * fmaf(t, d, U);
                S = t * f;
            }
            m = mn;
            const int out = own ? at : -1;  // one element of the maximum is left out
#pragma unroll
            for (int j = 0; j < PER_LANE; j++) add(j == out ? -INFINITY : x[j], m, S, U);
        } else {
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int j = 0; j < PER_LANE; j++) add(x[j], ref, S, U);
        }
        if (!p.alts) continue;
        least = lane_key(max(least, *(volatile Key*)&bound), 0);
        if (!__ballot(top >= value_of(least) && top > -INFINITY)) continue;
        // Elements above the list's last one are put in their places: the lanes' best ones, then the next ones of the
        // lanes that had one.
        find();
        auto best = [&]() {
            const Key k = key_of(top, from(piece(c, 0) + at / V * (64 * V)) + at % V);
            return top > -INFINITY ? k : 0;
        };
        Key mine = best();
        for (;;) {
            const unsigned long long can = __ballot(mine > least);
            if (!can) break;
            bool next;  // the lane's best is in the list, or not as good as what is
            if (p.alts > 1 && __popcll(can) > FEW) {
                list = first ? best16(mine, lane) : joined(list, best16(mine, lane), lane);
                const Key last = lane_key(list, p.alts - 1);
                next = mine && mine >= last;
                least = max(least, last);
            } else {  // one after the other, each before what it passes
                unsigned long long todo = p.alts > 1 ? can : 1ULL << best_lane(mine > least ? top : -INFINITY, mine);
                next = todo >> lane & 1;
                do {
                    const Key in = lane_key(mine, __ffsll(todo) - 1);
                    todo &= todo - 1;
                    if (in <= least) continue;
                    const Key before = moved<0x111>(list);
                    const int row16 = lane & 15, place = __popcll(__ballot(lane < 16 && list > in));
                    list = row16 < place ? list : row16 == place ? in : before;
                    least = max(least, lane_key(list, p.alts - 1));
                } while (todo);
            }
            first = false;
            float second = -INFINITY;
#pragma unroll
            for (int j = 0; j < PER_LANE; j++) {
                x[j] = next && j == at ? -INFINITY : x[j];
                second = fmaxf(second, x[j]);
            }
            top = next ? second : top;
            if (!__ballot(next && top >= value_of(least))) break;
            find();
            const Key k = best();
            mine = next ? k : mine;
        }
        if (lane == 0 && least > *(volatile Key*)&bound) bound = least;
    }
    S = wave_sum(S);
    U = wave_sum(U);
    const int words = HEAD + 2 * p.alts;
    // lane i: word i of the wave's part
    const float head = lane == 0 ? m : lane == 1 ? S : U;  // (and an unused word)
    if (splits == 1) {
        float* const part = lds + wave * words;
        if (lane < HEAD) part[lane] = head;
        if (lane < p.alts) *(Key*)(part + HEAD + 2 * lane) = list;
        __syncthreads();
    } else {
        float* const parts = p.work + JOIN_COUNTERS + (long)r * splits * 4 * words;
        float* const part = parts + (split * 4 + wave) * words;
        if (lane < HEAD) shared_store(part + lane, head);
        if (lane < p.alts)
            shared_store(part + HEAD + 2 * lane, __builtin_bit_cast(float, (unsigned)list), __builtin_bit_cast(float, (unsigned)(list >> 32)));
        if (!last_of((unsigned*)p.work + r, splits)) return;
        const int all = splits * 4 * words;
        for (int i0 = tid; i0 < all; i0 += 1024) {
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = shared_load(parts + min(i0 + 256 * k, all - 1));
#pragma unroll
            for (int k = 0; k < 4; k++) lds[min(i0 + 256 * k, all - 1)] = x[k];
        }
        __syncthreads();
    }
    Key best = 0;
    if (p.alts && splits == 1) {
        if (wave == 0) best = best_of_parts(lds, 4, p.alts, lane);
    } else if (p.alts) {
        best = best_of_parts(lds + wave * splits * words, splits, p.alts, lane);
        if (lane < 16) lists[wave * 16 + lane] = best;
        __syncthreads();
        best = best_of_rows(lists[lane], lane);
    }
    if (wave == 0) finish(p, r * p.out_stride + n, lds, 4 * splits, lane, tok, left_out ? -INFINITY : xt, best);
}

int score_splits(const MzScores& p) {
    const long chunks = (p.vocab + CHUNK - 1) / CHUNK, want = p.rows <= JOIN_COUNTERS ? 4L * mz_cu_count() / p.rows : 1;
    return (int)std::max(1L, std::min({want, (chunks + 3) / 4, (long)PARTS / 4}));
}

template <typename T>
hipError_t launch(hipStream_t s, const MzScores& p) {
    const int splits = score_splits(p);
    const dim3 grid((long)p.rows * splits);
    if (p.mask) hipLaunchKernelGGL((score_kernel<T, true>), grid, dim3(256), 0, s, p, splits);
    else hipLaunchKernelGGL((score_kernel<T, false>), grid, dim3(256), 0, s, p, splits);
    return hipGetLastError();
}

}  // namespace

size_t mz_scores_work(const MzScores& p) {
    const int splits = score_splits(p);
    return splits > 1 ? ((size_t)p.rows * splits * 4 * (HEAD + 2 * p.alts) + JOIN_COUNTERS) * 4 : 0;
}

hipError_t mz_scores_launch(hipStream_t s, const MzScores& p) { return p.half ? launch<f16>(s, p) : launch<float>(s, p); }
