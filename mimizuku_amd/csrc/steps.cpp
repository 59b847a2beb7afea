// C ABI: parts of a decoder step of a caller's own (mz_w4_*, mz_cross_attention, mz_sample): argument checks, and launches
// on the context's stream. What the device arrays hold (slots, lengths, settings) is checked by the kernels.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/mimizuku.h"
#include "mz_args.h"
#include "mz_internal.h"
#include "mz_kernels.h"

namespace {

constexpr int MAX_K = 1 << 24;
constexpr int64_t MAX_WEIGHTS = (int64_t)1 << 36;  // a wave packs 2048 of them: a launch has fewer than 2^32 threads along x
constexpr int MAX_POSITIONS = 1 << 30;         // (blocks of them are counted in 32 bits)
constexpr int MAX_SAMPLE_ROWS = (1 << 22) - 1;  // a workgroup of 1024 threads each: a launch has fewer than 2^32 along x

bool w4_shape_ok(int n, int k, int group) {
    return n > 0 && n <= MZ_W4_MOST_N && k > 0 && k <= MAX_K && k % 128 == 0 &&
           (int64_t)n * k <= MAX_WEIGHTS && (group == 32 || group == 64 || group == 128);
}

int check_w4(const char* who, const mz_w4* w, MzW4* out) {
    if (!w4_shape_ok(w->n, w->k, w->group))
        return mz_fail(MZ_ERR_ARG, "%s: %d x %d weights in groups of %d (k a multiple of 128, groups of 32, 64 or 128)", who, w->n, w->k, w->group);
    if (!w->codes || !w->scales || !aligned(w->codes, 16) || !aligned(w->scales, 16))
        return mz_fail(MZ_ERR_ARG, "%s: codes and scales must be multiples of 16 bytes", who);
    *out = {w->n, w->k, w->group, DP(unsigned char, w->codes), DP(f16, w->scales)};
    return MZ_OK;
}

// f16 [n][ld] weights to be packed, or unpacked to
int check_plain(const char* who, const mz_w4* w, uint64_t p, int64_t ld) {
    if (!p || !aligned(p, 16)) return mz_fail(MZ_ERR_ARG, "%s: the fp16 weights must be a multiple of 16 bytes", who);
    if (ld < w->k || ld % 8 || ld > MOST / w->n) return mz_fail(MZ_ERR_ARG, "%s: ld %lld of %d columns", who, (long long)ld, w->k);
    return MZ_OK;
}

int check_linear(const char* who, const mz_w4* w, const mz_w4_linear_args* a, MzW4* weights, MzW4Linear* out) {
    if (int r = check_w4(who, w, weights)) return r;
    const bool half = a->epilogue == MZ_EPI_F16 || a->epilogue == MZ_EPI_GELU_F16;
    if (!half && a->epilogue != MZ_EPI_RESID_F32 && a->epilogue != MZ_EPI_F32) return mz_fail(MZ_ERR_ARG, "%s: bad epilogue %d", who, a->epilogue);
    if (a->m < 0 || a->m > MZ_W4_MOST_M) return mz_fail(MZ_ERR_ARG, "%s: %d rows", who, a->m);
    const int64_t m = std::max(a->m, 1);
    if (!a->x || !aligned(a->x, 16) || a->ldx < w->k || a->ldx % 8 || a->ldx > MOST / m)
        return mz_fail(MZ_ERR_ARG, "%s: x must be a multiple of 16 bytes, ldx %lld one of 8 and at least %d", who, (long long)a->ldx, w->k);
    if (!a->out || !aligned(a->out, half ? 2 : 4) || !aligned(a->bias, 2) || a->ldo < w->n || a->ldo > MOST / m)
        return mz_fail(MZ_ERR_ARG, "%s: out and bias must be multiples of their elements' size, ldo %lld at least %d", who, (long long)a->ldo, w->n);
    *out = {a->epilogue, a->m, DP(const f16, a->x), (long)a->ldx, DP(const f16, a->bias), DP(void, a->out), (long)a->ldo};
    return MZ_OK;
}

int check_cross(const char* who, const mz_cross_attention_args* a, MzCross* out) {
    if (a->rows < 0 || a->tokens < 0 || a->slots < 0 || a->positions < 0 || a->positions > MAX_POSITIONS)
        return mz_fail(MZ_ERR_ARG, "%s: %d rows, %d tokens, %d slots, %d positions", who, a->rows, a->tokens, a->slots, a->positions);
    if (a->kv_heads <= 0 || a->heads <= 0 || a->heads % a->kv_heads || a->heads / a->kv_heads > 64)
        return mz_fail(MZ_ERR_ARG, "%s: %d query heads over %d", who, a->heads, a->kv_heads);
    if (!(a->scale > 0.f) || a->scale > 1048576.f) return mz_fail(MZ_ERR_ARG, "%s: scale %g", who, (double)a->scale);
    if (!a->q || !a->out || !aligned(a->q, 16) || !aligned(a->out, 16) || !aligned(a->k, 16) || !aligned(a->v, 16))
        return mz_fail(MZ_ERR_ARG, "%s: q, out, k and v must be multiples of 16 bytes", who);
    if ((!a->k || !a->v) && a->slots && a->positions) return mz_fail(MZ_ERR_ARG, "%s: null k or v", who);
    for (uint64_t p : {a->slot, a->count, a->first, a->len, a->lse, a->head_slot, a->align})
        if (!aligned(p, 4)) return mz_fail(MZ_ERR_ARG, "%s: addresses must be multiples of their elements' size", who);
    const int64_t n[3] = {a->rows, a->tokens, a->heads}, m[3] = {a->slots, a->positions, a->kv_heads};
    const int64_t qs[3] = {a->q_row, a->q_token, a->q_head}, os[3] = {a->out_row, a->out_token, a->out_head};
    const int64_t ks[3] = {a->k_slot, a->k_pos, a->k_head}, vs[3] = {a->v_slot, a->v_pos, a->v_head};
    if (!strides_ok(qs, n) || !strides_ok(os, n) || !strides_ok(ks, m) || !strides_ok(vs, m))
        return mz_fail(MZ_ERR_ARG, "%s: strides must be multiples of 8 elements, none negative", who);
    if (!apart(os, n)) return mz_fail(MZ_ERR_ARG, "%s: the output's rows overlap", who);
    if (a->align && (!a->head_slot || a->align_heads <= 0 || a->align_cols <= 0))
        return mz_fail(MZ_ERR_ARG, "%s: alignment rows need head_slot, align_heads and align_cols", who);
    if ((int64_t)a->rows * std::max(a->tokens, 1) > MOST / a->heads ||
        (a->align && (int64_t)a->rows * std::max(a->tokens, 1) > MOST / a->align_heads / a->align_cols))
        return mz_fail(MZ_ERR_ARG, "%s: too large", who);
    *out = {DP(const f16, a->q), DP(f16, a->out), (long)a->q_row, (long)a->q_token, (long)a->q_head, (long)a->out_row,
            (long)a->out_token, (long)a->out_head, DP(const f16, a->k), DP(const f16, a->v), (long)a->k_slot, (long)a->k_pos,
            (long)a->k_head, (long)a->v_slot, (long)a->v_pos, (long)a->v_head, a->rows, a->tokens, a->heads, a->kv_heads,
            a->slots, a->positions, a->scale, DP(const int, a->slot), DP(const int, a->count), DP(const int, a->first),
            DP(const int, a->len), DP(float, a->lse), a->align ? DP(const int, a->head_slot) : nullptr, DP(float, a->align),
            a->align_heads, a->align_cols, nullptr};
    if (!mz_cross_fits(*out)) return mz_fail(MZ_ERR_ARG, "%s: too large for one call", who);
    return MZ_OK;
}

int check_sample(const char* who, const mz_sample_args* a, MzSample* out) {
    if (a->dtype != MZ_DT_F16 && a->dtype != MZ_DT_F32) return mz_fail(MZ_ERR_ARG, "%s: bad dtype %d", who, a->dtype);
    if (a->rows < 0 || a->rows > MAX_SAMPLE_ROWS || a->vocab <= 0 || a->vocab > (1 << 30) || a->ld < a->vocab || a->ld > MOST / std::max(a->rows, 1))
        return mz_fail(MZ_ERR_ARG, "%s: %d rows of %d logits, ld %lld", who, a->rows, a->vocab, (long long)a->ld);
    if (!a->logits || !aligned(a->logits, a->dtype == MZ_DT_F32 ? 4 : 2))
        return mz_fail(MZ_ERR_ARG, "%s: logits must be a multiple of the element's size", who);
    for (uint64_t p : {a->temperatures, a->top_ps, a->min_ps, a->top_ks, a->u, a->tokens, a->logp, a->kept, a->at})
        if (!aligned(p, 4)) return mz_fail(MZ_ERR_ARG, "%s: addresses must be multiples of 4 bytes", who);
    if (!a->u || !a->tokens) return mz_fail(MZ_ERR_ARG, "%s: null u or tokens", who);
    if (!a->temperatures && !(a->temperature >= 0.f && std::isfinite(a->temperature)))
        return mz_fail(MZ_ERR_ARG, "%s: temperature %g", who, (double)a->temperature);
    if ((!a->top_ps && std::isnan(a->top_p)) || (!a->min_ps && std::isnan(a->min_p)))
        return mz_fail(MZ_ERR_ARG, "%s: top_p %g, min_p %g", who, (double)a->top_p, (double)a->min_p);
    if (a->stride < 1 || a->stride > MOST / std::max(a->rows, 1)) return mz_fail(MZ_ERR_ARG, "%s: stride %lld", who, (long long)a->stride);
    *out = {a->dtype == MZ_DT_F16, a->rows, a->vocab, DP(const void, a->logits), (long)a->ld, DP(const unsigned char, a->mask),
            a->temperature, a->top_p, a->min_p, a->top_k, DP(const float, a->temperatures), DP(const float, a->top_ps),
            DP(const float, a->min_ps), DP(const int, a->top_ks), DP(const float, a->u), DP(int, a->tokens), DP(float, a->logp),
            DP(int, a->kept), (long)a->stride, DP(const int, a->at), a->at_add};
    return MZ_OK;
}

}  // namespace

extern "C" int mz_w4_place(int n, int k, int group, uint64_t base, mz_w4* w, size_t* bytes) {
    if (w) *w = mz_w4{};
    if (bytes) *bytes = 0;
    if (!w4_shape_ok(n, k, group))
        return mz_fail(MZ_ERR_ARG, "mz_w4_place: %d x %d weights in groups of %d (k a multiple of 128, groups of 32, 64 or 128)", n, k, group);
    if (!aligned(base, 256)) return mz_fail(MZ_ERR_ARG, "mz_w4_place: base must be a multiple of 256 bytes");
    const uint64_t entries = ((uint64_t)n + 15) / 16 * (k / 128);  // tiles of 16 rows x 128 columns: 1024 bytes of codes
    if (w) *w = mz_w4{n, k, group, base, base + entries * 1024};
    if (bytes) *bytes = entries * 1024 + (entries * (16 * 128 / group) * 2 + 255) / 256 * 256;
    return MZ_OK;
}

extern "C" int mz_w4_pack(mz_ctx* c, const mz_w4* w, uint64_t src, int64_t ld) {
    if (!c || !w) return mz_fail(MZ_ERR_ARG, "mz_w4_pack: null argument");
    MzW4 weights;
    if (int r = check_w4("mz_w4_pack", w, &weights)) return r;
    if (int r = check_plain("mz_w4_pack", w, src, ld)) return r;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    return mz_hip(mz_w4_pack_launch(c->stream, weights, DP(const f16, src), (long)ld), "mz_w4_pack");
}

extern "C" int mz_w4_unpack(mz_ctx* c, const mz_w4* w, uint64_t dst, int64_t ld) {
    if (!c || !w) return mz_fail(MZ_ERR_ARG, "mz_w4_unpack: null argument");
    MzW4 weights;
    if (int r = check_w4("mz_w4_unpack", w, &weights)) return r;
    if (int r = check_plain("mz_w4_unpack", w, dst, ld)) return r;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    return mz_hip(mz_w4_unpack_launch(c->stream, weights, DP(f16, dst), (long)ld), "mz_w4_unpack");
}

extern "C" int mz_w4_linear(mz_ctx* c, const mz_w4* w, const mz_w4_linear_args* a) {
    if (!c || !w || !a) return mz_fail(MZ_ERR_ARG, "mz_w4_linear: null argument");
    MzW4 weights;
    MzW4Linear p;
    if (int r = check_linear("mz_w4_linear", w, a, &weights, &p)) return r;
    if (!a->m) return MZ_OK;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    return mz_hip(mz_w4_linear_launch(c->stream, weights, p), "mz_w4_linear");
}

extern "C" int mz_cross_attention_bytes(mz_ctx* c, const mz_cross_attention_args* a, size_t* bytes) {
    if (!c || !a || !bytes) return mz_fail(MZ_ERR_ARG, "mz_cross_attention_bytes: null argument");
    *bytes = 0;
    MzCross p;
    if (int r = check_cross("mz_cross_attention_bytes", a, &p)) return r;
    if (!a->rows || !a->tokens) return MZ_OK;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    *bytes = mz_cross_work(p);
    return MZ_OK;
}

extern "C" int mz_cross_attention(mz_ctx* c, const mz_cross_attention_args* a) {
    if (!c || !a) return mz_fail(MZ_ERR_ARG, "mz_cross_attention: null argument");
    MzCross p;
    if (int r = check_cross("mz_cross_attention", a, &p)) return r;
    if (!a->rows || !a->tokens) return MZ_OK;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    if (int r = check_work("mz_cross_attention", a->work, a->work_bytes, mz_cross_work(p))) return r;
    p.work = DP(float, a->work);
    return mz_hip(mz_cross_launch(c->stream, p), "mz_cross_attention");
}

extern "C" int mz_sample_bytes(mz_ctx* c, const mz_sample_args* a, size_t* bytes) {
    if (!c || !a || !bytes) return mz_fail(MZ_ERR_ARG, "mz_sample_bytes: null argument");
    *bytes = 0;
    MzSample p;
    return check_sample("mz_sample_bytes", a, &p);
}

extern "C" int mz_sample(mz_ctx* c, const mz_sample_args* a) {
    if (!c || !a) return mz_fail(MZ_ERR_ARG, "mz_sample: null argument");
    MzSample p;
    if (int r = check_sample("mz_sample", a, &p)) return r;
    if (!a->rows) return MZ_OK;
    OnDevice on(c->device);
    if (on.status()) return on.status();
    return mz_hip(mz_sample_launch(c->stream, p), "mz_sample");
}
