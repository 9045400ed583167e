"""Operators on device memory, for programs that run layers of their own over a session's states.

rms_norm, quantize_tokens, linear_i8 and CrossPlan.run call the entry points
of the same names in turbo_rocm.h, which say what each computes, what it
checks and how it runs. Their arrays are tensors on the context's GPU that
answer data_ptr(), shape, stride(), dtype and get_device() as torch's do (this
package imports no torch), or a `DeviceArray` over one of that GPU's buffers. Outputs are the caller's:
nothing is allocated.

`stream` is a HIP stream's handle (torch.cuda.current_stream().cuda_stream):
the work is enqueued there, behind the tensors' own, and the call returns at
once. Without it the call runs on the context's stream and waits, and what
other streams write into its arrays must be done before.
"""
import ctypes as C
import struct

from . import seam as S

ENQUEUE = 1   # TURBO_ROCM_ENQUEUE

_DTYPES = {"torch.float32": S.TURBO_DTYPE_F32, "torch.float16": S.TURBO_DTYPE_F16,
           "torch.bfloat16": S.TURBO_DTYPE_BF16, "torch.int8": S.TURBO_DTYPE_I8, "torch.uint8": S.TURBO_DTYPE_U8,
           "torch.int32": S.TURBO_DTYPE_I32}
_SIZES = {S.TURBO_DTYPE_F32: 4, S.TURBO_DTYPE_F16: 2, S.TURBO_DTYPE_BF16: 2, S.TURBO_DTYPE_I8: 1, S.TURBO_DTYPE_U8: 1,
          S.TURBO_DTYPE_I32: 4}
_known = {}   # dtype objects seen, and their TURBO_DTYPE codes


def dtype_code(dtype):
    """The TURBO_DTYPE code of a dtype: the code itself, torch's dtype or its name."""
    code = _known.get(dtype)
    if code is None:
        code = dtype if dtype in _SIZES else _DTYPES.get(str(dtype))
        if code is None:
            raise TypeError(f"{dtype} is no type of the operators' arrays")
        _known[dtype] = code
    return code


class DeviceArray:
    """An array in a buffer of the context's (Context.buffer: DEVICE, PINNED
    or SHARED; a session's output is one by Session.output): shape, and strides in elements (row after row by default),
    from `offset` bytes into it."""

    def __init__(self, buffer, shape, dtype, strides=None, offset=0):
        self.buffer, self.shape, self.dtype = buffer, tuple(shape), dtype_code(dtype)
        if strides is None:
            strides, n = [], 1
            for k in reversed(self.shape):
                strides.insert(0, n)
                n *= k
        self.strides = tuple(strides)
        if not 0 <= offset <= buffer.nbytes:
            raise ValueError(f"an array from byte {offset} of a buffer of {buffer.nbytes}")
        if not buffer.h:
            raise ValueError("an array of a buffer that is closed")
        h = S.turbo_native_handle()
        h.struct_size = C.sizeof(h)
        from . import _ok
        err = S.new_error()
        _ok(buffer.t.buffer_export(buffer.h, S.TURBO_HANDLE_CUDA_PTR, C.byref(h), C.byref(err)), err)
        self.address, self.bytes = h.handle + offset, buffer.nbytes - offset

    def data_ptr(self):
        return self.address

    def stride(self):
        return self.strides


# One turbo_rocm_tensor: data, bytes, shape[3], stride[2], ndim, dtype.
_ABSENT = (0,) * 9


def _tensor(t, device=None):
    # (device: the HIP device it has to be on, None without a context.)
    if t is None:
        return _ABSENT
    shape, stride = t.shape, t.stride()
    dtype = _known.get(t.dtype) or dtype_code(t.dtype)
    n = len(shape)
    # reach: what the strides reach, in elements (a tensor lies within its own storage).
    if n == 2:
        a, b = shape
        step, last = stride
        reach = (a - 1) * step + b if a and b else 0
        rest = a, b, 0, step, 0, 2, dtype
    elif n == 1:
        b, = shape
        last, = stride
        reach = b
        rest = b, 0, 0, 0, 0, 1, dtype
    elif n == 3:
        a, c, b = shape
        step, inner, last = stride
        reach = (a - 1) * step + (c - 1) * inner + b if a and c and b else 0
        rest = a, c, b, step, inner, 3, dtype
    else:
        raise ValueError(f"an array of {n} axes")
    if last != 1 and b > 1:
        raise ValueError("the last axis of an array must be contiguous")
    if type(t) is DeviceArray:
        if not t.buffer.h:
            raise ValueError("an array of a buffer that is closed")
        if device is not None and t.buffer.ctx.device != device:
            raise ValueError(f"an array on GPU {t.buffer.ctx.device}, not the context's {device}")
        return (t.address, t.bytes) + rest
    if device is None:
        if not t.is_cuda:
            raise ValueError("a tensor that is not on the GPU")
    elif t.get_device() != device:
        raise ValueError(f"a tensor that is not on GPU {device}, the context's")
    return (t.data_ptr(), reach * _SIZES[dtype]) + rest


_T = "QQQQQQQII"
_NORM = struct.Struct("=IIQd" + 7 * _T)
_CODES = struct.Struct("=IIQ" + 3 * _T)
_LINEAR = struct.Struct("=IIQ" + 6 * _T)
_CROSS = struct.Struct("=IIQQQd" + 5 * _T)


_functions = {}   # the library's, once looked up
_byref, _error, _ERROR = C.byref, S.turbo_error, C.sizeof(S.turbo_error)


def _handle(ctx):
    return (None, None) if ctx is None else (ctx.h, ctx.device)


def _on(stream):
    return (0, 0) if stream is None else (ENQUEUE, stream)


def _call(name, handle, packed):
    f = _functions.get(name)
    if f is None:
        from . import library
        f = _functions[name] = getattr(library(), name)
    err = _error()
    err.struct_size = _ERROR
    rc = f(handle, packed, _byref(err))
    if rc != S.TURBO_OK:
        from . import TurboError
        raise TurboError(rc, err.field, err.message.decode(errors="replace"))


def rms_norm(ctx, x, weight, eps, residual=None, sum=None, out=None, codes=None, scales=None, stream=None):
    """v = x (+ residual), y = v * weight / sqrt(mean(v^2) + eps): v into
    sum, y into out, y's int8 codes and scales into codes and scales."""
    h, on = _handle(ctx)
    _call("turbo_rocm_rms_norm", h,
          _NORM.pack(_NORM.size, *_on(stream), eps, *_tensor(x, on), *_tensor(residual, on), *_tensor(weight, on),
                     *_tensor(sum, on), *_tensor(out, on), *_tensor(codes, on), *_tensor(scales, on)))


def quantize_tokens(ctx, x, codes, scales, stream=None):
    """The int8 codes and scales of x's rows, as linear_i8 takes them."""
    h, on = _handle(ctx)
    _call("turbo_rocm_quantize_tokens", h,
          _CODES.pack(_CODES.size, *_on(stream), *_tensor(x, on), *_tensor(codes, on), *_tensor(scales, on)))


def linear_i8(ctx, codes, scales, weight, weight_scales, out, bias=None, stream=None):
    """out = (codes weight^T) * scales[:, None] * weight_scales + bias."""
    h, on = _handle(ctx)
    _call("turbo_rocm_linear_i8", h,
          _LINEAR.pack(_LINEAR.size, *_on(stream), *_tensor(codes, on), *_tensor(scales, on), *_tensor(weight, on),
                       *_tensor(weight_scales, on), *_tensor(bias, on), *_tensor(out, on)))


def _u32(values, what):
    # (ctypes would take a number's lowest 32 bits.)
    for x in values:
        if not 0 <= x < 1 << 32:
            raise ValueError(f"{what} of {x}")
    return values


def _lengths(q_lens, k_lens):
    n = len(q_lens)
    if len(k_lens) != n:
        raise ValueError(f"{n} query lengths and {len(k_lens)} key lengths")
    return (n, (C.c_uint32 * max(1, n))(*_u32(q_lens, "a query length")),
            (C.c_uint32 * max(1, n))(*_u32(k_lens, "a key length")))


def _cross_desc(q_lens, k_lens, heads, kv_heads, width, dtype):
    d = S.turbo_rocm_cross_desc()
    d.struct_size = C.sizeof(d)
    d.dtype = dtype_code(dtype)
    d.heads, d.kv_heads, d.width = _u32((heads, kv_heads, width), "heads or a width")
    d.batch, d.q_lens, d.k_lens = _lengths(q_lens, k_lens)
    return d


def _cross_call(q, k, v, out, mask, scale, workspace, stream, width, on=None):
    w, wn = (0, 0) if workspace is None else _tensor(workspace, on)[:2]
    return _CROSS.pack(_CROSS.size, *_on(stream), w, wn, max(1, width) ** -0.5 if scale is None else scale,
                       *_tensor(q, on), *_tensor(k, on), *_tensor(v, on), *_tensor(mask, on), *_tensor(out, on))


def check_cross(q_lens, k_lens, heads, kv_heads, width, dtype, q=None, k=None, v=None, out=None, mask=None, scale=None,
                stream=None):
    """A plan's and (with q) a call's checks without a device (turbo_rocm_cross_check)."""
    d = _cross_desc(q_lens, k_lens, heads, kv_heads, width, dtype)
    packed = None if q is None else _cross_call(q, k, v, out, mask, scale, None, stream, width)
    _call("turbo_rocm_cross_check", C.byref(d), packed)


def cross_cut(q_lens, k_lens, heads, kv_heads, width, dtype):
    """(rows, states) of a plan's largest workgroup (turbo_rocm_cross_cut); a test hook."""
    from . import _ok
    d = _cross_desc(q_lens, k_lens, heads, kv_heads, width, dtype)
    rows, states, err = C.c_uint32(), C.c_uint64(), S.new_error()
    _ok(_lib().turbo_rocm_cross_cut(C.byref(d), C.byref(rows), C.byref(states), C.byref(err)), err)
    return rows.value, states.value


def linear_i8_kernel(m, n, k, aligned):
    """The kernel of an int8 product (turbo_rocm_linear_i8_kernel); a test hook."""
    from . import _ok
    kernel, err = C.c_uint32(), S.new_error()
    _ok(_lib().turbo_rocm_linear_i8_kernel(m, n, k, 1 if aligned else 0, C.byref(kernel), C.byref(err)), err)
    return kernel.value


class CrossPlan:
    """Cross attention of sequences of these lengths (turbo_rocm_cross_plan_create)."""

    def __init__(self, ctx, q_lens, k_lens, heads, kv_heads, width, dtype):
        from . import _ok
        self.h = None
        self.ctx, self.width = ctx, width
        d = _cross_desc(q_lens, k_lens, heads, kv_heads, width, dtype)
        need, h = C.c_uint64(), C.c_void_p()
        err = S.new_error()
        _ok(_lib().turbo_rocm_cross_plan_create(None if ctx is None else ctx.h, C.byref(d), C.byref(need), C.byref(h),
                                                C.byref(err)), err)
        self.h, self.workspace_bytes = h, need.value

    def run(self, q, k, v, out, mask=None, scale=None, workspace=None, stream=None):
        """softmax(scale q k^T) v into out, per sequence and head over the
        states whose mask entry is not 0; scale 1 / sqrt(width) by default.
        workspace: a 1-d tensor (or DeviceArray) of workspace_bytes I8 or U8
        (none needed where that is 0), this call's own until it is done."""
        # (A plan works for as long as its context.)
        _call("turbo_rocm_cross_attention", self.h if self.ctx.h else None,
              _cross_call(q, k, v, out, mask, scale, workspace, stream, self.width, self.ctx.device))

    def close(self):
        if self.h:
            _lib().turbo_rocm_cross_plan_release(self.h)
            self.h = None


def _lib():
    from . import library
    return library()
