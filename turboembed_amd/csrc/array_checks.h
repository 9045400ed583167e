// The checks that the operators on device memory share (turbo_rocm.h): of a
// call's arrays, of what they may overlap, and how a call runs.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <mutex>
#include <string>
#include <utility>

#include "turbo_rocm.h"
#include "operators.h"
#include "session.h"

namespace rocm {

typedef turbo_rocm_tensor Tensor;
typedef unsigned __int128 u128;

inline uint32_t bit(uint32_t dtype) { return dtype < 32 ? 1u << dtype : 0u; }
inline const uint32_t F32 = bit(TURBO_DTYPE_F32), F16 = bit(TURBO_DTYPE_F16), BF16 = bit(TURBO_DTYPE_BF16),
               I8 = bit(TURBO_DTYPE_I8), I32 = bit(TURBO_DTYPE_I32), FLOATS = F32 | F16 | BF16;

inline uint64_t element(uint32_t dtype) { return dtype == TURBO_DTYPE_I8 ? 1 : bit(dtype) & (F16 | BF16) ? 2 : 4; }
inline Dt dt_of(uint32_t dtype) {
    return dtype == TURBO_DTYPE_F32 ? Dt::F32 : dtype == TURBO_DTYPE_F16 ? Dt::F16 : Dt::BF16;
}

[[noreturn]] inline void refuse(uint32_t field, const std::string &m) { fail(TURBO_E_INVALID_ARGUMENT, "rocm: " + m, field); }
[[noreturn]] inline void misshapen(uint32_t field, const std::string &m) { fail(TURBO_E_INVALID_SHAPE, "rocm: " + m, field); }

inline bool empty(const Tensor &t) {
    for (uint32_t i = 0; i < t.ndim; ++i)
        if (t.shape[i] == 0) return true;
    return false;
}

// Elements from the first to past the last.
inline u128 span(const Tensor &t) {
    if (empty(t)) return 0;
    u128 n = t.shape[t.ndim - 1];
    for (uint32_t i = 0; i + 1 < t.ndim; ++i) n += (u128)(t.shape[i] - 1) * t.stride[i];
    return n;
}

// An array of the call, absent or of ndim axes and one of the types; what its
// strides reach lies within its bytes.
struct Arg {
    const Tensor *t;
    const char *name;
    uint32_t field;
    bool given() const { return t->ndim != 0; }
};

inline void check_array(const Arg &a, uint32_t ndim, uint32_t types, bool optional) {
    const Tensor &t = *a.t;
    if (t.ndim == 0) {
        if (t.data || t.bytes) refuse(a.field, std::string(a.name) + " has an address but no axes");
        if (!optional) refuse(a.field, std::string(a.name) + " is not given");
        return;
    }
    if (t.ndim != ndim)
        misshapen(a.field, std::string(a.name) + " has " + std::to_string(t.ndim) + " axes, not " +
                               std::to_string(ndim));
    if (!(bit(t.dtype) & types))
        refuse(a.field, std::string(a.name) + " is of type " + std::to_string(t.dtype) + ", which it cannot be");
    // (An axis of 2^31 steps or more is past every kernel's index.)
    for (uint32_t i = 0; i < ndim; ++i)
        if (t.shape[i] > (uint64_t)INT32_MAX)
            misshapen(a.field, std::string(a.name) + "'s axis of " + std::to_string(t.shape[i]));
    if (empty(t)) return;
    if (!t.data) refuse(a.field, std::string(a.name) + " has no address");
    if (reinterpret_cast<uintptr_t>(t.data) % element(t.dtype))
        refuse(a.field, std::string(a.name) + " is not aligned to its elements");
    if (span(t) * element(t.dtype) > t.bytes)
        refuse(a.field, std::string(a.name) + " reaches past its " + std::to_string(t.bytes) + " bytes");
}

// No two elements of an output share a place: the axes one inside the other.
inline void check_apart(const Arg &a) {
    const Tensor &t = *a.t;
    if (!a.given() || empty(t) || t.ndim == 1) return;
    uint64_t shape[2] = {t.shape[0], t.ndim == 3 ? t.shape[1] : 1}, stride[2] = {t.stride[0], t.ndim == 3 ? t.stride[1] : 0};
    if (shape[1] > 1 && (shape[0] <= 1 || stride[1] > stride[0])) {
        std::swap(shape[0], shape[1]);
        std::swap(stride[0], stride[1]);
    }
    u128 width = t.shape[t.ndim - 1];
    for (int i = 1; i >= 0; --i) {
        if (shape[i] <= 1) continue;
        if (stride[i] < width) refuse(a.field, std::string(a.name) + "'s elements overlap");
        width += (u128)(shape[i] - 1) * stride[i];
    }
}

// t's bytes modulo `step`, where they are one run behind its first: of axes of
// multiples of it, and of `axes` shorter steps, `inner` the last. length 0: they
// are not.
struct Run {
    u128 length, inner = 0;
    int axes = 0;
};
inline Run run_within(const Tensor &t, u128 step) {
    Run r{t.shape[t.ndim - 1] * (u128)element(t.dtype)};
    for (uint32_t i = 0; i + 1 < t.ndim; ++i) {
        if (t.shape[i] == 1) continue;
        const u128 s = (u128)t.stride[i] * element(t.dtype);
        if (s >= step && s % step) return Run{0};
        if (s < step) r.length += (t.shape[i] - 1) * s, r.inner = s, ++r.axes;
    }
    return r.length <= step ? r : Run{0};
}

// Whether two arrays share a byte: their extents meet, unless they lie in
// different columns of rows of one length, which is a step of either, or of the
// rows within such a row (K and V side by side in a token's row, in a head's, or
// in a head's plane).
inline bool meet(const Tensor &a, const Tensor &b) {
    typedef __int128 i128;
    if (a.ndim == 0 || b.ndim == 0 || empty(a) || empty(b)) return false;
    const u128 a0 = reinterpret_cast<uintptr_t>(a.data), b0 = reinterpret_cast<uintptr_t>(b.data);
    const u128 a1 = a0 + span(a) * element(a.dtype), b1 = b0 + span(b) * element(b.dtype);
    if (a1 <= b0 || b1 <= a0) return false;
    const i128 wa = (i128)a.shape[a.ndim - 1] * element(a.dtype), wb = (i128)b.shape[b.ndim - 1] * element(b.dtype);
    // off: b's place in a's rows.
    const auto columns = [](i128 off, i128 step, i128 wa, i128 wb) {
        const i128 at = (off % step + step) % step;
        return at >= wa && at + wb <= step;
    };
    for (const Tensor *t : {&a, &b})
        for (uint32_t i = 0; i + 1 < t->ndim; ++i) {
            const i128 step = (i128)t->stride[i] * element(t->dtype);
            if (t->shape[i] == 1 || step == 0) continue;
            const Run ra = run_within(a, step), rb = run_within(b, step);
            if (!ra.length || !rb.length) continue;
            const i128 off = (((i128)b0 - (i128)a0) % step + step) % step, inner = ra.inner ? ra.inner : rb.inner;
            const auto clear = [&](i128 off) {   // of a's run, b's at off
                if (off >= (i128)ra.length || off + (i128)rb.length <= 0) return true;
                return inner && ra.axes < 2 && rb.axes < 2 && (!ra.axes || !rb.axes || ra.inner == rb.inner) &&
                       columns(off, inner, wa, wb);
            };
            if (clear(off) && clear(off - step)) return false;
        }
    return true;
}

inline bool same(const Tensor &a, const Tensor &b) {
    if (a.data != b.data || a.dtype != b.dtype) return false;
    for (uint32_t i = 0; i + 1 < a.ndim; ++i)
        if (a.shape[i] > 1 && a.stride[i] != b.stride[i]) return false;
    return true;
}

inline void check_clear(const Arg &out, const Arg &other, bool in_place = false) {
    if (!meet(*out.t, *other.t) || (in_place && same(*out.t, *other.t))) return;
    refuse(out.field, std::string(out.name) + " overlaps " + other.name);
}

inline void check_shape(const Arg &a, uint64_t n0, uint64_t n1, uint64_t n2 = 0) {
    const uint64_t want[3] = {n0, n1, n2};
    if (!a.given()) return;
    for (uint32_t i = 0; i < a.t->ndim; ++i)
        if (a.t->shape[i] != want[i])
            misshapen(a.field, std::string(a.name) + "'s axis " + std::to_string(i) + " is " +
                                   std::to_string(a.t->shape[i]) + ", not " + std::to_string(want[i]));
}

// The call's own fields, and how it runs: enqueued on the caller's stream, or
// on the context's and waited for.
template <class Call> void check_call(const Call *call) {
    if (!call) refuse(0, "no call");
    if (call->struct_size != sizeof(Call))
        fail(TURBO_E_INVALID_STRUCT_SIZE, "rocm: a call of " + std::to_string(call->struct_size) + " bytes, not " +
                                              std::to_string(sizeof(Call)));
    if (call->flags & ~TURBO_ROCM_ENQUEUE) refuse(0, "flags " + std::to_string(call->flags));
    if (!(call->flags & TURBO_ROCM_ENQUEUE) && call->stream) refuse(0, "a stream without TURBO_ROCM_ENQUEUE");
}

template <class Call, class Launch> void run_call(Context *c, const Call *call, const char *what, Launch &&launch) {
    if (!c) fail(TURBO_E_INVALID_HANDLE, "rocm: no context");
    OnDevice on(c->ordinal);
    if (call->flags & TURBO_ROCM_ENQUEUE) {
        hipStream_t s = static_cast<hipStream_t>(call->stream);
        if (s) {
            int device = -1;
            check(hipStreamGetDevice(s, &device), "the call's stream");
            if (device != c->ordinal)
                refuse(0, "a stream of device " + std::to_string(device) + ", not the context's " +
                              std::to_string(c->ordinal));
        }
        check(launch(s), what);
        return;
    }
    std::lock_guard<std::recursive_mutex> g(c->lock);
    // (Waited for even where a launch failed: one before it may be running.)
    const hipError_t launched = launch(c->stream), waited = hipStreamSynchronize(c->stream);
    check(launched, what);
    check(waited, what);
}

inline void *address(const Tensor &t) { return t.ndim == 0 || empty(t) ? nullptr : t.data; }

// A score's factor in base 2, as the kernels take it.
inline float base2(double scale) { return (float)(scale * 1.4426950408889634); }

}  // namespace rocm
