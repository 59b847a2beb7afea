// C ABI: key/value caches held in 8 bits (mz_kv8_*) and token scores (mz_token_scores): argument checks, and launches
// on the context's stream. What the device arrays hold (positions, lengths, slots, tokens) is checked by the kernels.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/mimizuku.h"
#include "mz_internal.h"
#include "mz_kernels.h"

#define DP(T, x) ((T*)(uintptr_t)(x))

namespace {

// The context's device is current while a call runs, whatever was before and will be after.
class OnDevice {
public:
    explicit OnDevice(int device) {
        if ((status_ = mz_hip(hipGetDevice(&before_), "hipGetDevice"))) return;
        if (before_ == device) before_ = -1;
        else status_ = mz_hip(hipSetDevice(device), "hipSetDevice");
    }
    ~OnDevice() {
        if (before_ >= 0) hipSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    int status() const { return status_; }

private:
    int before_ = -1, status_ = MZ_OK;
};

bool aligned(uint64_t p, uint64_t n) { return p % n == 0; }

// Elements of each tensor stay below this, so that no 64-bit byte offset of a kernel can wrap.
constexpr int64_t MOST = (int64_t)1 << 46;
constexpr int MAX_BLOCKS = (1 << 20) - 1;  // of a slot: its codes lie within 2^31 bytes, as far as a buffer descriptor reaches
constexpr int MAX_SCORE_ROWS = (1 << 24) - 1;  // a workgroup of 256 threads each: a launch has fewer than 2^32 along x

int check_cache(const char* who, const mz_kv8* kv, MzKv8* out) {
    if (kv->format != MZ_KV8_I8 && kv->format != MZ_KV8_E4M3) return mz_fail(MZ_ERR_ARG, "%s: bad cache format %d", who, kv->format);
    if (kv->slots <= 0 || kv->heads <= 0 || kv->blocks <= 0 || kv->blocks > MAX_BLOCKS ||
        (int64_t)kv->slots * kv->heads > MOST / MZ_KV_TILE / kv->blocks)
        return mz_fail(MZ_ERR_ARG, "%s: bad cache of %d slots, %d heads, %d blocks", who, kv->slots, kv->heads, kv->blocks);
    for (uint64_t p : {kv->k, kv->v, kv->k_open, kv->v_open})
        if (!p || !aligned(p, 16)) return mz_fail(MZ_ERR_ARG, "%s: cache addresses must be multiples of 16 bytes", who);
    for (uint64_t p : {kv->k_scale, kv->v_scale, kv->open})
        if (!p || !aligned(p, 4)) return mz_fail(MZ_ERR_ARG, "%s: cache addresses must be multiples of 4 bytes", who);
    *out = {kv->format, kv->slots, kv->heads, kv->blocks, DP(unsigned char, kv->k), DP(unsigned char, kv->v),
            DP(float, kv->k_scale), DP(float, kv->v_scale), DP(f16, kv->k_open), DP(f16, kv->v_open), DP(int, kv->open)};
    return MZ_OK;
}

// Offsets of rows x tokens x heads 64-channel rows: in range, and multiples of 8 elements.
bool strides_ok(const int64_t (&stride)[3], const int64_t (&n)[3]) {
    for (int i = 0; i < 3; i++)
        if (stride[i] < 0 || stride[i] % 8 || stride[i] > MOST || (n[i] > 1 && stride[i] > MOST / (n[i] - 1))) return false;
    return true;
}

// Whether those rows lie apart from each other, each dimension's steps outside what the smaller ones span.
bool apart(const int64_t (&stride)[3], const int64_t (&n)[3]) {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int a, int b) { return stride[a] < stride[b]; });
    int64_t span = 64;
    for (int i : order) {
        if (n[i] <= 1) continue;
        if (stride[i] < span) return false;
        span += stride[i] * (n[i] - 1);
    }
    return true;
}

int check_io(const char* who, const mz_kv8* kv, const mz_kv8_io* a, const MzKv8* cache, MzKv8Io* out) {
    if (a->rows < 0 || a->tokens < 0) return mz_fail(MZ_ERR_ARG, "%s: %d rows, %d tokens", who, a->rows, a->tokens);
    if (a->pos_stride < 0) return mz_fail(MZ_ERR_ARG, "%s: pos_stride %d", who, a->pos_stride);
    if (!aligned(a->k, 16) || !aligned(a->v, 16)) return mz_fail(MZ_ERR_ARG, "%s: k and v must be multiples of 16 bytes", who);
    if (!aligned(a->slot, 4) || !aligned(a->pos, 4) || !aligned(a->count, 4))
        return mz_fail(MZ_ERR_ARG, "%s: slot, pos and count must be multiples of 4 bytes", who);
    const int64_t stride[3] = {a->row_stride, a->token_stride, a->head_stride}, n[3] = {a->rows, a->tokens, kv->heads};
    if (!strides_ok(stride, n)) return mz_fail(MZ_ERR_ARG, "%s: strides must be multiples of 8 elements, none negative", who);
    *out = {DP(f16, a->k), DP(f16, a->v), (long)a->row_stride, (long)a->token_stride, (long)a->head_stride, a->rows,
            a->tokens, DP(int, a->slot), DP(int, a->pos), a->pos_stride, a->pos_add, DP(int, a->count)};
    if (!mz_kv8_io_fits(*cache, *out)) return mz_fail(MZ_ERR_ARG, "%s: too large for one call", who);
    return MZ_OK;
}

int check_attention(const char* who, const mz_kv8* kv, const mz_kv8_attention_args* a, MzKv8* cache, MzKv8Attn* out) {
    if (int r = check_cache(who, kv, cache)) return r;
    if (a->rows < 0 || a->tokens < 0) return mz_fail(MZ_ERR_ARG, "%s: %d rows, %d tokens", who, a->rows, a->tokens);
    if (a->heads <= 0 || a->heads % kv->heads || a->heads / kv->heads > 64)
        return mz_fail(MZ_ERR_ARG, "%s: %d query heads over a cache of %d", who, a->heads, kv->heads);
    if (!(a->scale > 0.f) || a->scale > 1048576.f) return mz_fail(MZ_ERR_ARG, "%s: scale %g", who, (double)a->scale);
    if (a->len_stride < 0) return mz_fail(MZ_ERR_ARG, "%s: len_stride %d", who, a->len_stride);
    if (!a->q || !a->out || !aligned(a->q, 16) || !aligned(a->out, 16))
        return mz_fail(MZ_ERR_ARG, "%s: q and out must be multiples of 16 bytes", who);
    for (uint64_t p : {a->slot, a->count, a->len, a->first, a->lse, a->head_slot, a->align})
        if (!aligned(p, 4)) return mz_fail(MZ_ERR_ARG, "%s: addresses must be multiples of their elements' size", who);
    const int64_t n[3] = {a->rows, a->tokens, a->heads};
    const int64_t qs[3] = {a->q_row, a->q_token, a->q_head}, os[3] = {a->out_row, a->out_token, a->out_head};
    if (!strides_ok(qs, n) || !strides_ok(os, n))
        return mz_fail(MZ_ERR_ARG, "%s: strides must be multiples of 8 elements, none negative", who);
    if (!apart(os, n)) return mz_fail(MZ_ERR_ARG, "%s: the output's rows overlap", who);
    if (a->align && (!a->head_slot || a->align_heads <= 0 || a->align_cols <= 0))
        return mz_fail(MZ_ERR_ARG, "%s: alignment rows need head_slot, align_heads and align_cols", who);
    if ((int64_t)a->rows * std::max(a->tokens, 1) > MOST / a->heads ||
        (a->align && (int64_t)a->rows * std::max(a->tokens, 1) > MOST / a->align_heads / a->align_cols))
        return mz_fail(MZ_ERR_ARG, "%s: too large", who);
    out->rows = a->rows;
    out->tokens = a->tokens;
    out->heads = a->heads;
    if (!mz_kv8_attn_fits(*cache, *out)) return mz_fail(MZ_ERR_ARG, "%s: too large for one call", who);
    *out = {DP(const f16, a->q), DP(f16, a->out), (long)a->q_row, (long)a->q_token, (long)a->q_head, (long)a->out_row,
            (long)a->out_token, (long)a->out_head, a->rows, a->tokens, a->heads, a->causal != 0, a->scale, DP(int, a->slot),
            DP(int, a->count), DP(int, a->len), a->len_stride, a->len_add, DP(int, a->first), DP(float, a->lse),
            a->align ? DP(int, a->head_slot) : nullptr, DP(float, a->align), a->align_heads, a->align_cols, nullptr};
    return MZ_OK;
}

int check_scores(const char* who, const mz_score_args* a, MzScores* out) {
    if (a->dtype != MZ_DT_F16 && a->dtype != MZ_DT_F32) return mz_fail(MZ_ERR_ARG, "%s: bad dtype %d", who, a->dtype);
    if (a->rows < 0 || a->rows > MAX_SCORE_ROWS || a->vocab <= 0 || a->vocab > (1 << 30) || a->ld < a->vocab || a->ld > MOST / std::max(a->rows, 1))
        return mz_fail(MZ_ERR_ARG, "%s: %d rows of %d logits, ld %lld", who, a->rows, a->vocab, (long long)a->ld);
    if (a->alts < 0 || a->alts > MZ_SCORE_ALTS) return mz_fail(MZ_ERR_ARG, "%s: %d alternatives (0 .. %d)", who, a->alts, MZ_SCORE_ALTS);
    if (!a->logits || !aligned(a->logits, a->dtype == MZ_DT_F32 ? 4 : 2))
        return mz_fail(MZ_ERR_ARG, "%s: logits must be a multiple of the element's size", who);
    for (uint64_t p : {a->tokens, a->at, a->logp, a->entropy, a->alt_ids, a->alt_logp})
        if (!aligned(p, 4)) return mz_fail(MZ_ERR_ARG, "%s: addresses must be multiples of 4 bytes", who);
    if (a->logp && !a->tokens) return mz_fail(MZ_ERR_ARG, "%s: logp needs tokens", who);
    // (results of different rows at different places)
    if (a->out_stride < 1 || a->out_stride > MOST / std::max(a->rows, 1) || a->token_stride < 0 ||
        a->token_stride > MOST / std::max(a->rows, 1))
        return mz_fail(MZ_ERR_ARG, "%s: token_stride %lld, out_stride %lld", who, (long long)a->token_stride, (long long)a->out_stride);
    *out = {a->dtype == MZ_DT_F16, a->rows, a->vocab, a->alts, DP(const void, a->logits), (long)a->ld,
            DP(const unsigned char, a->mask), DP(const int, a->tokens), (long)a->token_stride, DP(const int, a->at), a->at_add,
            DP(float, a->logp), DP(float, a->entropy), (long)a->out_stride, DP(int, a->alt_ids), DP(float, a->alt_logp), nullptr};
    return MZ_OK;
}

int check_work(const char* who, uint64_t work, size_t have, size_t need) {
    if (need && (!work || !aligned(work, 256) || have < need))
        return mz_fail(MZ_ERR_ARG, "%s: needs a workspace of %zu bytes, aligned to 256 (given %zu)", who, need, work ? have : (size_t)0);
    return MZ_OK;
}

}  // namespace

extern "C" int mz_kv8_place(int format, int slots, int heads, int max_tokens, uint64_t base, mz_kv8* kv, size_t* bytes) {
    if (kv) *kv = mz_kv8{};
    if (bytes) *bytes = 0;
    if (format != MZ_KV8_I8 && format != MZ_KV8_E4M3) return mz_fail(MZ_ERR_ARG, "mz_kv8_place: bad format %d", format);
    const int64_t blocks = ((int64_t)max_tokens + MZ_KV8_BLOCK - 1) / MZ_KV8_BLOCK;
    if (slots <= 0 || heads <= 0 || max_tokens <= 0 || blocks > MAX_BLOCKS || (int64_t)slots * heads > MOST / MZ_KV_TILE / blocks)
        return mz_fail(MZ_ERR_ARG, "mz_kv8_place: %d slots, %d heads, %d tokens", slots, heads, max_tokens);
    if (!aligned(base, 256)) return mz_fail(MZ_ERR_ARG, "mz_kv8_place: base must be a multiple of 256 bytes");
    const uint64_t sh = (uint64_t)slots * heads;
    uint64_t at = base;
    auto take = [&](uint64_t n) {
        const uint64_t r = at;
        at += (n + 255) & ~(uint64_t)255;
        return r;
    };
    mz_kv8 t{format, slots, heads, (int)blocks, 0, 0, 0, 0, 0, 0, 0};
    t.k = take(sh * blocks * MZ_KV_TILE);
    t.v = take(sh * blocks * MZ_KV_TILE);
    t.k_scale = take(sh * blocks * 4);
    t.v_scale = take(sh * blocks * 4);
    t.k_open = take(sh * MZ_KV_TILE * 2);
    t.v_open = take(sh * MZ_KV_TILE * 2);
    t.open = take(sh * 4);
    if (kv) *kv = t;
    if (bytes) *bytes = at - base;
    return MZ_OK;
}

extern "C" int mz_kv8_write(mz_ctx* c, const mz_kv8* kv, const mz_kv8_io* a) {
    if (!c || !kv || !a) return mz_fail(MZ_ERR_ARG, "mz_kv8_write: null argument");
    MzKv8 cache;
    MzKv8Io io;
    if (int r = check_cache("mz_kv8_write", kv, &cache)) return r;
    if (int r = check_io("mz_kv8_write", kv, a, &cache, &io)) return r;
    if (!a->rows || !a->tokens) return MZ_OK;
    if (!a->k || !a->v) return mz_fail(MZ_ERR_ARG, "mz_kv8_write: null k or v");
    OnDevice on(c->device);
    if (on.status()) return on.status();
    return mz_hip(mz_kv8_write_launch(c->stream, cache, io), "mz_kv8_write");
}

extern "C" int mz_kv8_read(mz_ctx* c, const mz_kv8* kv, const mz_kv8_io* a) {
    if (!c || !kv || !a) return mz_fail(MZ_ERR_ARG, "mz_kv8_read: null argument");
    MzKv8 cache;
    MzKv8Io io;
    if (int r = check_cache("mz_kv8_read", kv, &cache)) return r;
    if (int r = check_io("mz_kv8_read", kv, a, &cache, &io)) return r;
    const int64_t stride[3] = {a->row_stride, a->token_stride, a->head_stride}, n[3] = {a->rows, a->tokens, kv->heads};
    if (!apart(stride, n)) return mz_fail(MZ_ERR_ARG, "mz_kv8_read: the rows read into overlap");
    if (!a->rows || !a->tokens || (!a->k && !a->v)) return MZ_OK;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    return mz_hip(mz_kv8_read_launch(c->stream, cache, io), "mz_kv8_read");
}

extern "C" int mz_kv8_attention_bytes(mz_ctx* c, const mz_kv8* kv, const mz_kv8_attention_args* a, size_t* bytes) {
    if (!c || !kv || !a || !bytes) return mz_fail(MZ_ERR_ARG, "mz_kv8_attention_bytes: null argument");
    *bytes = 0;
    MzKv8 cache;
    MzKv8Attn p;
    if (int r = check_attention("mz_kv8_attention_bytes", kv, a, &cache, &p)) return r;
    if (!a->rows || !a->tokens) return MZ_OK;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    *bytes = mz_kv8_attn_work(cache, p);
    return MZ_OK;
}

extern "C" int mz_kv8_attention(mz_ctx* c, const mz_kv8* kv, const mz_kv8_attention_args* a) {
    if (!c || !kv || !a) return mz_fail(MZ_ERR_ARG, "mz_kv8_attention: null argument");
    MzKv8 cache;
    MzKv8Attn p;
    if (int r = check_attention("mz_kv8_attention", kv, a, &cache, &p)) return r;
    if (!a->rows || !a->tokens) return MZ_OK;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    if (int r = check_work("mz_kv8_attention", a->work, a->work_bytes, mz_kv8_attn_work(cache, p))) return r;
    p.work = DP(float, a->work);
    return mz_hip(mz_kv8_attn_launch(c->stream, cache, p), "mz_kv8_attention");
}

extern "C" int mz_token_scores_bytes(mz_ctx* c, const mz_score_args* a, size_t* bytes) {
    if (!c || !a || !bytes) return mz_fail(MZ_ERR_ARG, "mz_token_scores_bytes: null argument");
    *bytes = 0;
    MzScores p;
    if (int r = check_scores("mz_token_scores_bytes", a, &p)) return r;
    if (!a->rows) return MZ_OK;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    *bytes = mz_scores_work(p);
    return MZ_OK;
}

extern "C" int mz_token_scores(mz_ctx* c, const mz_score_args* a) {
    if (!c || !a) return mz_fail(MZ_ERR_ARG, "mz_token_scores: null argument");
    MzScores p;
    if (int r = check_scores("mz_token_scores", a, &p)) return r;
    if (!a->rows) return MZ_OK;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    if (int r = check_work("mz_token_scores", a->work, a->work_bytes, mz_scores_work(p))) return r;
    p.work = DP(float, a->work);
    return mz_hip(mz_scores_launch(c->stream, p), "mz_token_scores");
}
