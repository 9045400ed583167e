// A cache of states in pages, and the attention of a call's own tokens
// (turbo_rocm.h): checks and entry points. The kernels are in cache_rows.hip
// and self_tiles.h.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "array_checks.h"
#include "cache.h"

using namespace rocm;

namespace rocm {

namespace {

// Rows (tokens times heads), a cache's slots and the positions of a sequence's
// pages are numbered in 31 bits, with room for a tile past the last.
constexpr uint64_t MOST = 1u << 30;

void check_heads(const Arg &a, uint64_t heads, uint64_t kv, uint64_t width) {
    if (width == 0 || width > 128)
        misshapen(a.field, std::string(a.name) + "'s heads are " + std::to_string(width) + " wide, not 1 to 128");
    if (heads == 0 || kv == 0 || heads % kv)
        misshapen(a.field, std::to_string(heads) + " heads over " + std::to_string(kv) + " key heads");
    const uint64_t tokens = a.t->shape[0];
    if ((u128)tokens * heads > MOST)
        fail(TURBO_E_CAPACITY, "rocm: " + std::to_string(tokens) + " tokens of " + std::to_string(heads) +
                                   " heads in one call", a.field);
}

// starts, [sequences + 1]: the number of sequences.
uint64_t check_starts(const Arg &starts) {
    check_array(starts, 1, I32, false);
    if (starts.t->shape[0] == 0) misshapen(starts.field, "starts has no entry");
    return starts.t->shape[0] - 1;
}

// The cache's arrays as a call has them, field its first one's place.
struct CacheArrays {
    Arg k, v, ks, vs, starts, lengths, pages;
    CacheArrays(const turbo_rocm_cache &c, uint32_t field)
        : k{&c.k, "the cache's k", field}, v{&c.v, "the cache's v", field + 1}, ks{&c.k_scales, "k_scales", field + 2},
          vs{&c.v_scales, "v_scales", field + 3}, starts{&c.starts, "starts", field + 4},
          lengths{&c.lengths, "lengths", field + 5}, pages{&c.pages, "pages", field + 6} {}
};

// A call's cache, for rows of the type `own` and the shape [., kv, width].
// written: its states are an output.
CacheArgs check_cache(const turbo_rocm_cache &c, uint32_t field, uint32_t own, uint64_t kv, uint64_t width,
                      uint64_t tokens, bool written) {
    const CacheArrays a(c, field);
    if (c.reserved) refuse(0, "the cache's reserved field is not 0");
    if (c.page_tokens == 0 || c.page_tokens > MOST) refuse(0, "pages of " + std::to_string(c.page_tokens) + " tokens");
    check_array(a.k, 3, own | I8, false);
    const bool i8 = c.k.dtype == TURBO_DTYPE_I8;
    check_array(a.v, 3, bit(c.k.dtype), false);
    const uint64_t slots = c.k.shape[0];
    if (slots > MOST) fail(TURBO_E_CAPACITY, "rocm: a cache of " + std::to_string(slots) + " slots", a.k.field);
    for (const Arg &s : {a.k, a.v}) check_shape(s, slots, kv, width);
    for (const Arg &s : {a.ks, a.vs}) {
        check_array(s, 2, F32, !i8);
        if (!i8 && s.given()) refuse(s.field, std::string(s.name) + " of states that are not I8");
        check_shape(s, slots, kv);
    }
    const uint64_t seqs = check_starts(a.starts);
    check_array(a.lengths, 1, I32, false);
    check_shape(a.lengths, seqs, 0);
    check_array(a.pages, 2, I32, false);
    if (a.pages.t->shape[0] != seqs) check_shape(a.pages, seqs, a.pages.t->shape[1]);
    const uint64_t columns = a.pages.t->shape[1];
    if ((u128)columns * c.page_tokens > MOST)
        fail(TURBO_E_CAPACITY, "rocm: " + std::to_string(columns) + " pages of " + std::to_string(c.page_tokens) +
                                   " tokens for a sequence", a.pages.field);
    if (written) {
        const Arg outs[] = {a.k, a.v, a.ks, a.vs};
        for (int i = 0; i < 4; ++i) {
            check_apart(outs[i]);
            for (int j = 0; j < i; ++j) check_clear(outs[i], outs[j]);
            for (const Arg &in : {a.starts, a.lengths, a.pages}) check_clear(outs[i], in);
        }
    }
    CacheArgs r{};
    r.k = address(c.k), r.v = address(c.v);
    r.k_scales = static_cast<float *>(address(c.k_scales)), r.v_scales = static_cast<float *>(address(c.v_scales));
    for (int i = 0; i < 2; ++i) r.ks[i] = c.k.stride[i], r.vs[i] = c.v.stride[i];
    r.kss = c.k_scales.stride[0], r.vss = c.v_scales.stride[0];
    r.starts = static_cast<const int32_t *>(address(c.starts));
    r.lengths = static_cast<const int32_t *>(address(c.lengths));
    r.pages = static_cast<const int32_t *>(address(c.pages));
    r.page_row = c.pages.stride[0], r.paged = true;
    r.seqs = (int)seqs, r.columns = (int)columns, r.page_tokens = (int)c.page_tokens;
    r.page_count = (int)(slots / c.page_tokens);
    if (r.page_count == 0) r.columns = 0;   // no page, no position
    r.tokens = (int)tokens, r.kv = (int)kv, r.width = (int)width;
    return r;
}

// The rows of a call that move to or from a cache; into: from the cache.
template <class Call> void move(Context *c, const Call *call, const char *what, bool into) {
    check_call(call);
    const Arg k{&call->k, "k", 1}, v{&call->v, "v", 2};
    check_array(k, 3, FLOATS, false);
    const uint32_t own = bit(call->k.dtype);
    check_array(v, 3, own, false);
    const uint64_t tokens = call->k.shape[0], kv = call->k.shape[1], width = call->k.shape[2];
    check_heads(k, kv, kv, width);
    check_shape(v, tokens, kv, width);
    CacheArgs a = check_cache(call->cache, 3, own, kv, width, tokens, !into);
    const CacheArrays h(call->cache, 3);
    if (into) {
        check_apart(k), check_apart(v), check_clear(v, k);
        for (const Arg &o : {k, v})
            for (const Arg &i : {h.k, h.v, h.ks, h.vs, h.starts, h.lengths, h.pages}) check_clear(o, i);
    } else {
        for (const Arg &o : {h.k, h.v, h.ks, h.vs})
            for (const Arg &i : {k, v}) check_clear(o, i);
    }
    const bool i8 = call->cache.k.dtype == TURBO_DTYPE_I8;
    const Dt t = dt_of(call->k.dtype);
    run_call(c, call, what, [&](hipStream_t s) {
        const uint64_t ks[2] = {call->k.stride[0], call->k.stride[1]}, vs[2] = {call->v.stride[0], call->v.stride[1]};
        return into ? cache_read(s, a, t, i8, address(call->k), address(call->v), ks, vs)
                    : cache_write(s, a, t, i8, address(call->k), address(call->v), ks, vs);
    });
}

void check_scale(double scale) {
    if (!std::isfinite(base2(scale))) refuse(0, "scale must be finite, in F32");
}

// What the two attentions' arguments have in common.
void attend(SelfArgs &a, const Tensor &q, const Tensor &out, double scale, uint32_t window, uint64_t heads) {
    a.q = address(q), a.out = address(out);
    for (int i = 0; i < 2; ++i) a.qs[i] = q.stride[i], a.os[i] = out.stride[i];
    a.dt = dt_of(q.dtype);
    a.share = (int)(heads / a.c.kv);
    a.window = window == 0 || window > (uint32_t)INT32_MAX ? INT32_MAX : (int)window;
    a.scale = base2(scale);
    a.turn = a.scale > 0 ? 1.0f : a.scale < 0 ? -1.0f : 0.0f;
    a.scale = a.scale == 0 ? 1.0f : std::fabs(a.scale);
}

void prompt(Context *c, const turbo_rocm_prompt_attention_call *call) {
    check_call(call);
    const Arg q{&call->q, "q", 1}, k{&call->k, "k", 2}, v{&call->v, "v", 3}, starts{&call->starts, "starts", 4},
        out{&call->out, "out", 5};
    if (call->reserved) refuse(0, "the call's reserved field is not 0");
    check_scale(call->scale);
    check_array(q, 3, FLOATS, false);
    const uint32_t own = bit(call->q.dtype);
    check_array(k, 3, own, false);
    check_array(v, 3, own, false);
    check_array(out, 3, own, false);
    const uint64_t tokens = call->q.shape[0], heads = call->q.shape[1], kv = call->k.shape[1], width = call->q.shape[2];
    check_heads(q, heads, kv, width);
    for (const Arg &s : {k, v}) check_shape(s, tokens, kv, width);
    check_shape(out, tokens, heads, width);
    const uint64_t seqs = check_starts(starts);
    check_apart(out);
    for (const Arg &i : {q, k, v, starts}) check_clear(out, i);
    SelfArgs a{};
    a.c.k = address(call->k), a.c.v = address(call->v);
    for (int i = 0; i < 2; ++i) a.c.ks[i] = call->k.stride[i], a.c.vs[i] = call->v.stride[i];
    a.c.starts = static_cast<const int32_t *>(address(call->starts));
    a.c.seqs = (int)seqs, a.c.tokens = (int)tokens, a.c.kv = (int)kv, a.c.width = (int)width;
    attend(a, call->q, call->out, call->scale, call->window, heads);
    const SelfLaunch f = self_plan(a);
    run_call(c, call, "prompt_attention", [&](hipStream_t s) { return self_attention(s, a, f); });
}

void cached(Context *c, const turbo_rocm_cache_attention_call *call) {
    check_call(call);
    const Arg q{&call->q, "q", 1}, out{&call->out, "out", 2};
    if (call->reserved) refuse(0, "the call's reserved field is not 0");
    check_scale(call->scale);
    check_array(q, 3, FLOATS, false);
    const uint32_t own = bit(call->q.dtype);
    check_array(out, 3, own, false);
    const uint64_t tokens = call->q.shape[0], heads = call->q.shape[1], width = call->q.shape[2];
    const uint64_t kv = call->cache.k.ndim == 3 ? call->cache.k.shape[1] : 0;
    if (kv) check_heads(q, heads, kv, width);   // (check_cache says what is wrong with the array)
    check_shape(out, tokens, heads, width);
    SelfArgs a{};
    a.c = check_cache(call->cache, 3, own, kv, width, tokens, false);
    if (!kv) check_heads(q, heads, kv, width);
    const CacheArrays h(call->cache, 3);
    check_apart(out);
    for (const Arg &i : {q, h.k, h.v, h.ks, h.vs, h.starts, h.lengths, h.pages}) check_clear(out, i);
    a.i8 = call->cache.k.dtype == TURBO_DTYPE_I8;
    attend(a, call->q, call->out, call->scale, call->window, heads);
    const uint64_t need = self_workspace(tokens, (uint64_t)a.c.seqs, (int)heads, (int)kv, (int)width);
    if (call->workspace_bytes < need || (need && !call->workspace))
        fail(TURBO_E_CAPACITY, "rocm: a workspace of " + std::to_string(call->workspace_bytes) + " bytes, not " +
                                   std::to_string(need));
    if (reinterpret_cast<uintptr_t>(call->workspace) % 16) refuse(0, "the workspace is not 16-byte aligned");
    if (need) {
        Tensor ws{};
        ws.data = call->workspace, ws.bytes = need, ws.shape[0] = need, ws.ndim = 1, ws.dtype = TURBO_DTYPE_I8;
        for (const Arg &i : {q, out, h.k, h.v, h.ks, h.vs, h.starts, h.lengths, h.pages})
            check_clear(i, Arg{&ws, "the workspace", 0});
    }
    a.ws = static_cast<float *>(call->workspace);
    const SelfLaunch f = self_plan(a);
    run_call(c, call, "cache_attention", [&](hipStream_t s) { return self_attention(s, a, f); });
}

}  // namespace
}  // namespace rocm

extern "C" {

int32_t turbo_rocm_prompt_attention(void *ctx, const turbo_rocm_prompt_attention_call *call, turbo_error *err) {
    return guarded(err, [&] {
        prompt(static_cast<Context *>(ctx), call);
        return TURBO_OK;
    });
}

int32_t turbo_rocm_cache_attention(void *ctx, const turbo_rocm_cache_attention_call *call, turbo_error *err) {
    return guarded(err, [&] {
        cached(static_cast<Context *>(ctx), call);
        return TURBO_OK;
    });
}

int32_t turbo_rocm_cache_write(void *ctx, const turbo_rocm_cache_rows_call *call, turbo_error *err) {
    return guarded(err, [&] {
        move(static_cast<Context *>(ctx), call, "cache_write", false);
        return TURBO_OK;
    });
}

int32_t turbo_rocm_cache_read(void *ctx, const turbo_rocm_cache_rows_call *call, turbo_error *err) {
    return guarded(err, [&] {
        move(static_cast<Context *>(ctx), call, "cache_read", true);
        return TURBO_OK;
    });
}

int32_t turbo_rocm_cache_workspace(uint64_t tokens, uint64_t sequences, uint32_t heads, uint32_t kv_heads,
                                   uint32_t width, uint32_t dtype, uint64_t *bytes, turbo_error *err) {
    return guarded(err, [&] {
        if (!bytes) refuse(0, "nowhere to leave the bytes");
        if (!(bit(dtype) & FLOATS)) fail(TURBO_E_INVALID_ENUM, "rocm: cache attention of type " + std::to_string(dtype));
        if (sequences > (uint64_t)INT32_MAX) misshapen(0, std::to_string(sequences) + " sequences");
        Tensor q{};
        q.shape[0] = tokens;
        check_heads(Arg{&q, "q", 0}, heads, kv_heads, width);
        *bytes = self_workspace(tokens, sequences, (int)heads, (int)kv_heads, (int)width);
        return TURBO_OK;
    });
}

int32_t turbo_rocm_self_kernel(uint64_t tokens, uint64_t sequences, uint32_t heads, uint32_t kv_heads, uint32_t width,
                               uint32_t dtype, uint32_t states, uint32_t aligned, uint32_t *rows, uint32_t *waves,
                               uint32_t *held, turbo_error *err) {
    return guarded(err, [&] {
        if (!rows || !waves || !held) refuse(0, "nowhere to leave the kernel");
        if (!(bit(dtype) & FLOATS)) fail(TURBO_E_INVALID_ENUM, "rocm: attention of type " + std::to_string(dtype));
        if (states > 2) refuse(0, "states " + std::to_string(states));
        if (tokens == 0 || sequences == 0 || sequences > (uint64_t)INT32_MAX)
            misshapen(0, std::to_string(tokens) + " tokens of " + std::to_string(sequences) + " sequences");
        Tensor q{};
        q.shape[0] = tokens;
        check_heads(Arg{&q, "q", 0}, heads, kv_heads, width);
        SelfArgs a{};
        a.c.k = a.c.v = reinterpret_cast<void *>((uintptr_t)(aligned ? 16 : 4));
        a.c.seqs = (int)sequences, a.c.tokens = (int)tokens, a.c.kv = (int)kv_heads, a.c.width = (int)width;
        a.c.paged = states != 0, a.c.columns = a.c.page_tokens = 1;
        a.i8 = states == 2, a.dt = dt_of(dtype), a.share = (int)(heads / kv_heads);
        const SelfLaunch f = self_plan(a);
        *rows = (uint32_t)f.rows, *waves = f.rows == 128 || f.split ? 4 : 1, *held = (uint32_t)f.held;
        return TURBO_OK;
    });
}

}  // extern "C"
