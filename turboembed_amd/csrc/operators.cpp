// The operators on device memory (turbo_rocm.h): their checks and entry
// points. The kernels are in row_codes.hip, linear_i8.hip and
// cross_attention.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "array_checks.h"

using namespace rocm;

namespace rocm {

namespace {

// ---- rms_norm and quantize_tokens ------------------------------------------------

void check_rows(const Arg &x) {
    if (x.t->shape[1] > ROW_COLS_MAX)
        misshapen(x.field, "rows of " + std::to_string(x.t->shape[1]) + " values, past " + std::to_string(ROW_COLS_MAX));
}

void rms_norm(Context *c, const turbo_rocm_rms_norm_call *call) {
    check_call(call);
    const Arg x{&call->x, "x", 1}, res{&call->residual, "residual", 2}, w{&call->weight, "weight", 3},
        sum{&call->sum, "sum", 4}, out{&call->out, "out", 5}, codes{&call->codes, "codes", 6},
        scales{&call->scales, "scales", 7};
    if (!std::isfinite(call->eps) || call->eps <= 0) refuse(0, "eps must be positive and finite");
    check_array(x, 2, FLOATS, false);
    const uint32_t own = bit(x.t->dtype);
    check_array(res, 2, own | F32, true);
    check_array(w, 1, own | F32, false);
    const uint32_t rt = res.given() ? res.t->dtype : x.t->dtype;
    if (sum.given() && !res.given()) refuse(sum.field, "sum without a residual");
    check_array(sum, 2, bit(rt), true);
    check_array(out, 2, FLOATS, true);
    check_array(codes, 2, I8, true);
    check_array(scales, 1, F32, true);
    if (codes.given() != scales.given()) refuse(codes.given() ? scales.field : codes.field, "codes and scales go together");
    if (!out.given() && !codes.given()) refuse(out.field, "neither out nor codes is given");
    const uint64_t rows = x.t->shape[0], cols = x.t->shape[1];
    check_rows(x);
    for (const Arg &a : {res, sum, out, codes}) check_shape(a, rows, cols);
    check_shape(w, cols, 0);
    check_shape(scales, rows, 0);
    const Arg outs[] = {sum, out, codes, scales};
    for (int i = 0; i < 4; ++i) {
        check_apart(outs[i]);
        check_clear(outs[i], x, i < 2);
        check_clear(outs[i], res, i == 0);
        check_clear(outs[i], w);
        for (int j = 0; j < i; ++j) check_clear(outs[i], outs[j]);
    }
    RowArgs a{};
    a.x = address(*x.t), a.res = address(*res.t), a.w = address(*w.t);
    a.sum = address(*sum.t), a.out = address(*out.t);
    a.codes = static_cast<int8_t *>(address(*codes.t)), a.scales = static_cast<float *>(address(*scales.t));
    a.ldx = x.t->stride[0], a.ldr = res.t->stride[0], a.lds = sum.t->stride[0], a.ldo = out.t->stride[0];
    a.ldc = codes.t->stride[0];
    a.xt = dt_of(x.t->dtype), a.rt = dt_of(rt), a.wt = dt_of(w.t->dtype), a.ot = dt_of(out.t->dtype);
    a.rows = (int)rows, a.cols = (int)cols, a.eps = call->eps;
    run_call(c, call, "rms_norm", [&](hipStream_t s) { return row_codes(s, a); });
}

void quantize_tokens(Context *c, const turbo_rocm_quantize_tokens_call *call) {
    check_call(call);
    const Arg x{&call->x, "x", 1}, codes{&call->codes, "codes", 2}, scales{&call->scales, "scales", 3};
    check_array(x, 2, FLOATS, false);
    check_array(codes, 2, I8, false);
    check_array(scales, 1, F32, false);
    check_rows(x);
    check_shape(codes, x.t->shape[0], x.t->shape[1]);
    check_shape(scales, x.t->shape[0], 0);
    for (const Arg &o : {codes, scales}) {
        check_apart(o);
        check_clear(o, x);
    }
    check_clear(scales, codes);
    RowArgs a{};
    a.x = address(*x.t), a.ldx = x.t->stride[0];
    a.codes = static_cast<int8_t *>(address(*codes.t)), a.ldc = codes.t->stride[0];
    a.scales = static_cast<float *>(address(*scales.t));
    a.xt = a.rt = dt_of(x.t->dtype);
    a.rows = (int)x.t->shape[0], a.cols = (int)x.t->shape[1];
    run_call(c, call, "quantize_tokens", [&](hipStream_t s) { return row_codes(s, a); });
}

// ---- linear_i8 -----------------------------------------------------------------------

void linear(Context *c, const turbo_rocm_linear_i8_call *call) {
    check_call(call);
    const Arg codes{&call->codes, "codes", 1}, scales{&call->scales, "scales", 2}, weight{&call->weight, "weight", 3},
        wscales{&call->weight_scales, "weight_scales", 4}, bias{&call->bias, "bias", 5}, out{&call->out, "out", 6};
    check_array(codes, 2, I8, false);
    check_array(scales, 1, F32, false);
    check_array(weight, 2, I8, false);
    check_array(wscales, 1, F32, false);
    check_array(bias, 1, F32, true);
    check_array(out, 2, FLOATS, false);
    const uint64_t m = codes.t->shape[0], k = codes.t->shape[1], n = weight.t->shape[0];
    if (k > I8_INNER_MAX)
        misshapen(codes.field, "an inner width of " + std::to_string(k) + ", past " + std::to_string(I8_INNER_MAX));
    check_shape(scales, m, 0);
    check_shape(weight, n, k);
    check_shape(wscales, n, 0);
    check_shape(bias, n, 0);
    check_shape(out, m, n);
    check_apart(out);
    for (const Arg &i : {codes, scales, weight, wscales, bias}) check_clear(out, i);
    LinearArgs a{};
    a.a = static_cast<const int8_t *>(address(*codes.t)), a.lda = codes.t->stride[0];
    a.w = static_cast<const int8_t *>(address(*weight.t)), a.ldw = weight.t->stride[0];
    a.as = static_cast<const float *>(address(*scales.t)), a.ws = static_cast<const float *>(address(*wscales.t));
    a.bias = static_cast<const float *>(address(*bias.t));
    a.out = address(*out.t), a.ldo = out.t->stride[0], a.ot = dt_of(out.t->dtype);
    a.m = (int)m, a.n = (int)n, a.k = (int)k;
    run_call(c, call, "linear_i8", [&](hipStream_t s) { return linear_i8(s, a); });
}

// ---- cross_attention -------------------------------------------------------------

struct CrossPlan {
    Context *ctx = nullptr;
    int ordinal = 0;   // (the context's, which may be gone when the plan is released)
    uint32_t dtype = 0, heads = 0, kv = 0, width = 0;
    uint64_t tokens = 0, states = 0, workspace = 0;
    int items = 0, joins = 0, part_rows = 0, most_rows = 0;
    bool one_wave = true;
    uint64_t parts = 0;
    DevPtr work;   // the items, then the joins
};

struct Totals {
    uint64_t tokens = 0, states = 0;
};

Totals check_desc(const turbo_rocm_cross_desc *d) {
    if (!d) refuse(0, "no description");
    if (d->struct_size != sizeof *d)
        fail(TURBO_E_INVALID_STRUCT_SIZE, "rocm: a description of " + std::to_string(d->struct_size) + " bytes, not " +
                                              std::to_string(sizeof *d));
    if (!(bit(d->dtype) & FLOATS)) fail(TURBO_E_INVALID_ENUM, "rocm: cross attention of type " + std::to_string(d->dtype));
    if (d->heads == 0 || d->kv_heads == 0 || d->heads % d->kv_heads)
        refuse(0, std::to_string(d->heads) + " heads over " + std::to_string(d->kv_heads) + " key heads");
    if (d->width == 0 || d->width > 128) refuse(0, "a head width of " + std::to_string(d->width) + ", not 1 to 128");
    if (d->batch && (!d->q_lens || !d->k_lens)) refuse(0, "no lengths");
    Totals t;
    for (uint32_t i = 0; i < d->batch; ++i) t.tokens += d->q_lens[i], t.states += d->k_lens[i];
    // (Rows and states are numbered in 31 bits.)
    if ((u128)t.tokens * d->heads > (u128)INT32_MAX || t.states > (uint64_t)INT32_MAX)
        fail(TURBO_E_CAPACITY, "rocm: " + std::to_string(t.tokens) + " tokens of " + std::to_string(d->heads) +
                                   " heads and " + std::to_string(t.states) + " states in one plan");
    return t;
}

void check_cross(const turbo_rocm_cross_attention_call *call, uint32_t dtype, uint32_t heads, uint32_t kv,
                 uint32_t width, const Totals &n) {
    check_call(call);
    const Arg q{&call->q, "q", 1}, k{&call->k, "k", 2}, v{&call->v, "v", 3}, mask{&call->mask, "mask", 4},
        out{&call->out, "out", 5};
    if (!std::isfinite(base2(call->scale))) refuse(0, "scale must be finite, in F32");
    for (const Arg &a : {q, k, v, out}) {
        check_array(a, 3, bit(dtype), false);
        const bool states = a.field == 2 || a.field == 3;
        check_shape(a, a.t->shape[0], states ? kv : heads, width);
        if (a.t->shape[0] < (states ? n.states : n.tokens))
            misshapen(a.field, std::string(a.name) + " has " + std::to_string(a.t->shape[0]) +
                                   " rows, fewer than the plan's");
    }
    check_array(mask, 1, I32, true);
    if (mask.given() && mask.t->shape[0] < n.states)
        misshapen(mask.field, "mask has " + std::to_string(mask.t->shape[0]) + " entries, fewer than the plan's states");
    check_apart(out);
    for (const Arg &a : {q, k, v, mask}) check_clear(out, a);
}

// How a plan's rows and keys are cut: row blocks of 32 (a wave) or 128 (four),
// and runs of at most `slice` keys. The choice is the least of an estimate of
// the call's time in us, fitted to what 23 calls took (F16, BF16 and F32, widths
// 32 to 128, 1 to 2048 rows a sequence) at 14 cuts each: its choice is within 9%
// of the best of the 14 for all but one (20%). The terms:
// - a compute unit's time for 64 keys of an item among others: products and
//   softmax, or its keys and values from memory (20.6 KB/us a unit), or the
//   caches where several row blocks read them (42 KB/us); a part's way to
//   memory and back beside it;
// - the longest item's time when it runs alone, of which the last items leave
//   a quarter;
// - the join's launch.
struct Cut {
    int rows;
    uint64_t slice;
};
Cut choose_cut(const turbo_rocm_cross_desc &d) {
    const uint64_t share = d.heads / d.kv_heads;
    uint64_t longest = 0;
    for (uint32_t s = 0; s < d.batch; ++s) longest = std::max<uint64_t>(longest, d.k_lens[s]);
    const bool f32 = d.dtype == TURBO_DTYPE_F32;
    const double dp = (d.width + 31) / 32 * 32, bytes = 128.0 * d.width * (f32 ? 4 : 2);
    Cut best{128, std::max<uint64_t>(64, longest)};
    double least = INFINITY;
    for (int rows : {32, 128}) {
        const double wave = f32 ? 0.045 * dp : 0.33 + 0.0077 * dp, work = rows == 32 ? wave / 2.6 : wave;
        const double alone = f32 ? 0.076 * dp : rows == 32 ? 0.97 + 0.0046 * dp : 0.57 + 0.0064 * dp;
        const double fixed = f32 && rows == 32 ? 2.8 : 0.36;   // (few such waves a unit: little beside its start)
        for (uint64_t slice = 64;; slice *= 2) {
            double total = 0, most = 0;
            bool joined = false;
            for (uint32_t s = 0; s < d.batch; ++s) {
                const uint64_t r = d.q_lens[s] * share, blocks = (r + rows - 1) / rows;
                if (!blocks) continue;
                const uint64_t pieces = std::max<uint64_t>(1, (d.k_lens[s] + slice - 1) / slice);
                const double tiles = std::ceil((double)d.k_lens[s] / pieces / 64);
                const double part = pieces > 1 ? 8.0 * std::min<uint64_t>(r, rows) * (d.width + 2) / 14800 : 0;
                total += (double)(blocks * d.kv_heads * pieces) *
                         (fixed + part + tiles * std::max(work, bytes / (blocks > 1 ? 42200 : 20600)));
                most = std::max(most, tiles * alone + 2.6);
                joined |= pieces > 1;
            }
            const double time = std::max(total / 256 + 0.25 * most, most) + (joined ? 6.1 : 0);
            if (time < least) least = time, best = {rows, slice};
            if (slice >= longest) break;
        }
    }
    return best;
}

// The items of a plan, in the order of their workgroups, and the joins.
void lay_out(const turbo_rocm_cross_desc &d, std::vector<CrossItem> &items, std::vector<CrossJoin> &joins,
             int &part_rows, uint64_t &parts) {
    const uint64_t share = d.heads / d.kv_heads;
    const Cut cut = choose_cut(d);
    part_rows = cut.rows;
    const uint64_t slice = cut.slice;
    // (A launch holds less than 2^32 threads.)
    u128 workgroups = 0;
    for (uint32_t s = 0; s < d.batch; ++s)
        workgroups += (u128)((d.q_lens[s] * share + part_rows - 1) / part_rows) * d.kv_heads *
                      std::max<uint64_t>(1, (d.k_lens[s] + slice - 1) / slice);
    if (workgroups > 1u << 23)
        fail(TURBO_E_CAPACITY, "rocm: a plan of " + std::to_string((uint64_t)workgroups) + " workgroups, past 2^23");

    // The row blocks of a (sequence, key head) read the same keys: they go to
    // one XCD (workgroups go to the 8 in turn), the XCD with the least work so
    // far, the longest first.
    struct Group {
        uint32_t seq, kv;
        uint64_t q0, k0, work;
    };
    std::vector<Group> groups;
    uint64_t q0 = 0, k0 = 0;
    for (uint32_t s = 0; s < d.batch; ++s) {
        const uint64_t rows = d.q_lens[s] * share;
        for (uint32_t h = 0; h < d.kv_heads && rows; ++h)
            groups.push_back({s, h, q0, k0, (rows + part_rows - 1) / part_rows * (d.k_lens[s] + 64ull)});
        q0 += d.q_lens[s], k0 += d.k_lens[s];
    }
    std::stable_sort(groups.begin(), groups.end(), [](const Group &a, const Group &b) { return a.work > b.work; });
    constexpr int XCDS = 8;
    std::vector<CrossItem> lists[XCDS];
    uint64_t load[XCDS] = {};
    parts = 0;
    for (const Group &g : groups) {
        const int x = (int)(std::min_element(load, load + XCDS) - load);
        load[x] += g.work;
        const uint64_t rows = d.q_lens[g.seq] * share, nk = d.k_lens[g.seq];
        const uint64_t cuts = std::max<uint64_t>(1, (nk + slice - 1) / slice);
        // Equal runs, whole 64s but for the last.
        const uint64_t run = (nk + cuts * 64 - 1) / (cuts * 64) * 64;
        for (uint64_t r = 0; r < rows; r += part_rows) {
            CrossItem it{};
            it.q0 = (int32_t)g.q0, it.kv = (int32_t)g.kv;
            it.row0 = (int32_t)r, it.rows = (int32_t)std::min<uint64_t>(part_rows, rows - r);
            const uint64_t pieces = run ? (nk + run - 1) / run : 1;
            if (pieces > 1)
                joins.push_back({it.q0, it.row0, it.rows, it.kv, (int32_t)parts, (int32_t)pieces, {0, 0}});
            for (uint64_t i = 0; i < pieces; ++i) {
                it.k0 = (int32_t)(g.k0 + i * run);
                it.nk = (int32_t)std::min(run, nk - i * run);
                it.part = pieces > 1 ? (int32_t)parts++ : -1;
                lists[x].push_back(it);
            }
        }
    }
    size_t total = 0, taken[XCDS] = {};
    for (const auto &l : lists) total += l.size();
    items.reserve(total);
    for (int x = 0; items.size() < total; x = (x + 1) % XCDS) {
        int from = x;
        if (taken[x] == lists[x].size())   // a list at its end: from the one with the most left
            for (int y = 0; y < XCDS; ++y)
                if (lists[y].size() - taken[y] > lists[from].size() - taken[from]) from = y;
        items.push_back(lists[from][taken[from]++]);
    }
}

CrossPlan *cross_plan_create(Context *c, const turbo_rocm_cross_desc *d) {
    const Totals t = check_desc(d);
    if (!c) fail(TURBO_E_INVALID_HANDLE, "rocm: no context");
    auto p = std::make_unique<CrossPlan>();
    p->ctx = c, p->ordinal = c->ordinal;
    p->dtype = d->dtype, p->heads = d->heads, p->kv = d->kv_heads, p->width = d->width;
    p->tokens = t.tokens, p->states = t.states;
    std::vector<CrossItem> items;
    std::vector<CrossJoin> joins;
    lay_out(*d, items, joins, p->part_rows, p->parts);
    for (const CrossItem &it : items) p->one_wave &= it.rows <= 32;
    for (const CrossJoin &j : joins) p->most_rows = std::max(p->most_rows, j.rows);
    p->workspace = p->parts * cross_part_floats(p->most_rows, (int)d->width) * 4;
    p->items = (int)items.size(), p->joins = (int)joins.size();
    const size_t ib = items.size() * sizeof(CrossItem), jb = joins.size() * sizeof(CrossJoin);
    if (ib + jb) {
        std::lock_guard<std::recursive_mutex> g(c->lock);
        OnDevice on(c->ordinal);
        p->work.reset(dev_alloc(ib + jb, "a cross attention plan"));
        check(hipMemcpyAsync(p->work.get(), items.data(), ib, hipMemcpyHostToDevice, c->stream), "a cross attention plan");
        if (jb)
            check(hipMemcpyAsync((char *)p->work.get() + ib, joins.data(), jb, hipMemcpyHostToDevice, c->stream),
                  "a cross attention plan");
        check(hipStreamSynchronize(c->stream), "a cross attention plan");
    }
    return p.release();
}

void cross_run(CrossPlan *p, const turbo_rocm_cross_attention_call *call) {
    if (!p) {
        check_call(call);
        fail(TURBO_E_INVALID_HANDLE, "rocm: no plan");
    }
    check_cross(call, p->dtype, p->heads, p->kv, p->width, Totals{p->tokens, p->states});
    if (call->workspace_bytes < p->workspace || (p->workspace && !call->workspace))
        fail(TURBO_E_CAPACITY, "rocm: a workspace of " + std::to_string(call->workspace_bytes) + " bytes, not " +
                                   std::to_string(p->workspace));
    if (reinterpret_cast<uintptr_t>(call->workspace) % 16) refuse(0, "the workspace is not 16-byte aligned");
    if (p->workspace) {
        Tensor ws{};
        ws.data = call->workspace, ws.bytes = p->workspace, ws.shape[0] = p->workspace, ws.ndim = 1;
        ws.dtype = TURBO_DTYPE_I8;
        const Arg arrays[] = {{&call->q, "q", 1}, {&call->k, "k", 2}, {&call->v, "v", 3}, {&call->mask, "mask", 4},
                              {&call->out, "out", 5}};
        for (const Arg &a : arrays) check_clear(a, Arg{&ws, "the workspace", 0});
    }
    CrossArgs a{};
    a.q = address(call->q), a.k = address(call->k), a.v = address(call->v), a.out = address(call->out);
    a.mask = static_cast<const int32_t *>(address(call->mask));
    a.ws = static_cast<float *>(call->workspace);
    a.items = static_cast<const CrossItem *>(p->work.get());
    a.joins = reinterpret_cast<const CrossJoin *>(a.items + p->items);
    for (int i = 0; i < 2; ++i)
        a.qs[i] = call->q.stride[i], a.ks[i] = call->k.stride[i], a.vs[i] = call->v.stride[i],
        a.os[i] = call->out.stride[i];
    a.dt = dt_of(p->dtype);
    a.n_items = p->items, a.n_joins = p->joins, a.part_rows = p->part_rows, a.most_rows = p->most_rows;
    a.one_wave = p->one_wave;
    a.share = (int)(p->heads / p->kv), a.width = (int)p->width;
    a.scale = base2(call->scale);
    a.turn = a.scale > 0 ? 1.0f : a.scale < 0 ? -1.0f : 0.0f;
    a.scale = a.scale == 0 ? 1.0f : std::fabs(a.scale);
    run_call(p->ctx, call, "cross_attention", [&](hipStream_t s) { return cross_attention(s, a); });
}

}  // namespace
}  // namespace rocm

extern "C" {

int32_t turbo_rocm_context_device(void *ctx, uint32_t *device, turbo_error *err) {
    return guarded(err, [&] {
        if (!ctx) fail(TURBO_E_INVALID_HANDLE, "rocm: no context");
        if (!device) refuse(0, "nowhere to leave the device");
        *device = (uint32_t)static_cast<Context *>(ctx)->ordinal;
        return TURBO_OK;
    });
}

int32_t turbo_rocm_cross_plan_create(void *ctx, const turbo_rocm_cross_desc *desc, uint64_t *workspace_bytes,
                                     void **out, turbo_error *err) {
    return guarded(err, [&] {
        if (!out) refuse(0, "nowhere to leave the plan");
        CrossPlan *p = cross_plan_create(static_cast<Context *>(ctx), desc);
        if (workspace_bytes) *workspace_bytes = p->workspace;
        *out = p;
        return TURBO_OK;
    });
}

void turbo_rocm_cross_plan_release(void *plan) {
    if (!plan) return;
    CrossPlan *p = static_cast<CrossPlan *>(plan);
    OnDevice on(p->ordinal);
    delete p;   // (hipFree waits for the device's work.)
}

int32_t turbo_rocm_cross_attention(void *plan, const turbo_rocm_cross_attention_call *call, turbo_error *err) {
    return guarded(err, [&] {
        cross_run(static_cast<CrossPlan *>(plan), call);
        return TURBO_OK;
    });
}

int32_t turbo_rocm_cross_check(const turbo_rocm_cross_desc *desc, const turbo_rocm_cross_attention_call *call,
                               turbo_error *err) {
    return guarded(err, [&] {
        const Totals t = check_desc(desc);
        if (call) check_cross(call, desc->dtype, desc->heads, desc->kv_heads, desc->width, t);
        return TURBO_OK;
    });
}

int32_t turbo_rocm_linear_i8_kernel(uint32_t m, uint32_t n, uint32_t k, uint32_t aligned, uint32_t *kernel,
                                    turbo_error *err) {
    return guarded(err, [&] {
        if (!kernel) refuse(0, "nowhere to leave the kernel");
        if (m == 0 || n == 0 || m > (uint32_t)INT32_MAX || n > (uint32_t)INT32_MAX || k > I8_INNER_MAX)
            misshapen(0, "a product of " + std::to_string(m) + " x " + std::to_string(n) + " x " + std::to_string(k));
        *kernel = k < 16 ? 0 : (uint32_t)linear_i8_kernel((int)m, (int)n, (int)k, aligned != 0);
        return TURBO_OK;
    });
}

int32_t turbo_rocm_cross_cut(const turbo_rocm_cross_desc *desc, uint32_t *rows, uint64_t *states, turbo_error *err) {
    return guarded(err, [&] {
        check_desc(desc);
        if (!rows || !states) refuse(0, "nowhere to leave the cut");
        const Cut cut = choose_cut(*desc);
        *rows = (uint32_t)cut.rows, *states = cut.slice;
        return TURBO_OK;
    });
}

int32_t turbo_rocm_rms_norm(void *ctx, const turbo_rocm_rms_norm_call *call, turbo_error *err) {
    return guarded(err, [&] {
        rms_norm(static_cast<Context *>(ctx), call);
        return TURBO_OK;
    });
}

int32_t turbo_rocm_quantize_tokens(void *ctx, const turbo_rocm_quantize_tokens_call *call, turbo_error *err) {
    return guarded(err, [&] {
        quantize_tokens(static_cast<Context *>(ctx), call);
        return TURBO_OK;
    });
}

int32_t turbo_rocm_linear_i8(void *ctx, const turbo_rocm_linear_i8_call *call, turbo_error *err) {
    return guarded(err, [&] {
        linear(static_cast<Context *>(ctx), call);
        return TURBO_OK;
    });
}

}  // extern "C"
