"""The operators' handles and arrays on a device: arrays of another device, of closed buffers and on the host, and
plans that outlive their contexts, are refused before any kernel."""
import ctypes as C

import pytest
import torch

import turboembed_amd as T
from turboembed_amd import seam as S

pytestmark = pytest.mark.gpu


class Elsewhere:
    """A tensor's twin that says it is on another GPU: nothing may read it."""
    def __init__(self, t):
        self.t, self.shape, self.dtype = t, t.shape, t.dtype

    def data_ptr(self):
        return self.t.data_ptr()

    def stride(self):
        return self.t.stride()

    def get_device(self):
        return 7


def _norm(context, **kw):
    a = dict(x=torch.ones(3, 40, device="cuda"), weight=torch.ones(40, device="cuda"), eps=1e-6,
             out=torch.full((3, 40), 5.0, device="cuda"))
    a.update(kw)
    torch.cuda.synchronize()
    context.rms_norm(**a)
    return a["out"]


def test_a_context_names_its_device(context):
    assert context.device == torch.cuda.current_device()
    device = C.c_uint32(99)
    err = S.new_error()
    assert T.library().turbo_rocm_context_device(None, C.byref(device), C.byref(err)) == S.TURBO_E_INVALID_HANDLE
    assert T.library().turbo_rocm_context_device(context.h, None, C.byref(err)) == S.TURBO_E_INVALID_ARGUMENT
    assert device.value == 99


@pytest.mark.parametrize("name", ["x", "weight", "out"])
def test_an_array_of_another_device_is_refused(context, name):
    arrays = dict(x=torch.ones(3, 40, device="cuda"), weight=torch.ones(40, device="cuda"),
                  out=torch.full((3, 40), 5.0, device="cuda"))
    for wrong in (Elsewhere(arrays[name]), arrays[name].cpu()):
        with pytest.raises(ValueError, match="GPU 0"):
            _norm(context, **{**arrays, name: wrong})
    assert (arrays["out"] == 5).all()


def test_a_workspace_of_another_device_is_refused(context):
    plan = context.cross_plan((1,), (4096,), 1, 1, 64, S.TURBO_DTYPE_F16)
    assert plan.workspace_bytes > 0
    q, k = torch.zeros(1, 1, 64, device="cuda").half(), torch.zeros(4096, 1, 64, device="cuda").half()
    ws = torch.zeros(plan.workspace_bytes, device="cuda", dtype=torch.int8)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="GPU 0"):
        plan.run(q, k, k, torch.empty_like(q), workspace=Elsewhere(ws))
    plan.close()


def test_an_array_of_a_closed_buffer_is_refused(context):
    buf = context.buffer(480)
    x = T.DeviceArray(buf, (3, 40), S.TURBO_DTYPE_F32)
    for offset in (-4, 484):
        with pytest.raises(ValueError):
            T.DeviceArray(buf, (1,), S.TURBO_DTYPE_F32, offset=offset)
    buf.view()[:] = 0
    assert (_norm(context, x=x) == 0).all()
    buf.close()
    with pytest.raises(ValueError, match="closed"):
        _norm(context, x=x)


def test_a_plan_after_its_context(runtime):
    ctx = runtime.context(0)
    q, k = torch.ones(2, 3, 16, device="cuda"), torch.ones(5, 3, 16, device="cuda")
    out = torch.full_like(q, 5.0)
    plan = ctx.cross_plan((2,), (5,), 3, 3, 16, torch.float32)
    assert plan.workspace_bytes == 0
    torch.cuda.synchronize()
    plan.run(q, k, k, out)
    assert (out == 1).all()
    out.fill_(5.0)
    torch.cuda.synchronize()
    ctx.close()
    with pytest.raises(T.TurboError) as e:
        plan.run(q, k, k, out)
    assert e.value.code == S.TURBO_E_INVALID_HANDLE and (out == 5).all()
    with pytest.raises(T.TurboError) as e:
        ctx.rms_norm(q[0], q[0, 0], 1e-6, out=out[0])
    assert e.value.code == S.TURBO_E_INVALID_HANDLE
    plan.close()


def test_calls_at_once_from_threads(context):
    """One plan and one context, every thread on a stream of its own with its own arrays, or waiting on the
    context's: each gets what it gets alone."""
    import threading
    plan = context.cross_plan((3, 1), (2100, 700), 4, 2, 64, torch.float16)
    assert plan.workspace_bytes > 0
    kv = torch.randn(2800, 2, 2, 64, generator=torch.Generator().manual_seed(0)).half().cuda()
    w = torch.randint(-127, 128, (80, 256), generator=torch.Generator().manual_seed(1), dtype=torch.int8).cuda()
    ones = torch.ones(256, device="cuda")

    def arrays(seed):
        q = torch.randn(4, 4, 64, generator=torch.Generator().manual_seed(seed)).half().cuda()
        return dict(q=q, o=torch.zeros_like(q), c=torch.zeros(4, 256, dtype=torch.int8, device="cuda"),
                    s=torch.zeros(4, device="cuda"), y=torch.zeros(4, 80, device="cuda"),
                    ws=torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda"))

    def layer(a, stream):
        plan.run(a["q"], kv[:, 0], kv[:, 1], a["o"], workspace=a["ws"], stream=stream)
        context.rms_norm(a["o"].view(4, 256), ones, 1e-6, codes=a["c"], scales=a["s"], stream=stream)
        context.linear_i8(a["c"], a["s"], w, ones[:80], a["y"], stream=stream)
    sets = [arrays(10 + i) for i in range(6)]
    torch.cuda.synchronize()
    want = []
    for a in sets:
        layer(a, None)
        want.append({k: a[k].clone() for k in "ocsy"})
    torch.cuda.synchronize()
    failures = []

    def work(i):
        try:
            stream = torch.cuda.Stream() if i % 3 else None
            for _ in range(20):
                if stream is None:
                    layer(sets[i], None)
                else:
                    layer(sets[i], stream.cuda_stream)
            if stream is not None:
                stream.synchronize()
            assert all(torch.equal(sets[i][k], want[i][k]) for k in "ocsy")
        except Exception as e:   # noqa: BLE001
            failures.append((i, e))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures, failures
    plan.close()


@pytest.mark.parametrize("waits", [False, True])
def test_an_error_of_the_caller_s_own_is_the_caller_s(context, waits):
    """A HIP call of the program's has failed on this thread, and nobody has asked why yet: an operator after it says
    how its own launches went, and leaves the program its error."""
    lib = T.library()
    x, w = torch.randn(3, 256, device="cuda"), torch.ones(256, device="cuda")
    y, c, s = torch.zeros(3, 256, device="cuda"), torch.zeros(3, 256, dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda")
    w8, o = torch.ones(40, 256, dtype=torch.int8, device="cuda"), torch.zeros(3, 40, device="cuda")
    k = torch.randn(2000, 4, 64, device="cuda")
    a = torch.zeros(3, 4, 64, device="cuda")
    plan = context.cross_plan((3,), (2000,), 4, 4, 64, torch.float32)
    assert plan.workspace_bytes > 0     # (two launches)
    ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda")
    stream = None if waits else torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()

    def calls():
        context.rms_norm(x, w, 1e-6, out=y, stream=stream)
        context.quantize_tokens(x, c, s, stream=stream)
        context.linear_i8(c, s, w8, w[:40], o, stream=stream)
        plan.run(x.view(3, 4, 64), k, k, a, workspace=ws, stream=stream)
    try:
        wrong = lib.hipSetDevice(4096)
        assert wrong != 0 and lib.hipPeekAtLastError() == wrong
        calls()
        assert lib.hipPeekAtLastError() == wrong
    finally:
        lib.hipGetLastError()
    torch.cuda.synchronize()
    got = [t.clone() for t in (y, c, s, o, a)]
    calls()
    torch.cuda.synchronize()
    assert all(torch.equal(g, t) and (g != 0).any() for g, t in zip(got, (y, c, s, o, a)))
    plan.close()


def test_a_session_s_states_without_a_copy(context):
    """A range for each token: the run's output is the tokens' states, read by the operators where it lies."""
    import numpy as np
    import small
    desc = small.bert(seed=5, hidden=96, heads=3, inter=64)
    model = context.load(desc)
    s = model.session(3, 24, S.TURBO_PRECISION_EXACT, max_ranges=72)
    with pytest.raises(T.TurboError) as e:
        s.output()
    assert e.value.code == S.TURBO_E_INVALID_STATE
    ids = np.random.Generator(np.random.PCG64(1)).integers(3, desc.vocab_size - 1, size=(3, 24)).astype(np.int32)
    lens = [24, 7, 15]
    mask = (np.arange(24)[None] < np.array(lens)[:, None]).astype(np.int32)
    s.write_ranges(ids, mask, [(r, i, i + 1) for r in range(3) for i in range(lens[r])], normalize=S.TURBO_NORMALIZE_NONE)
    s.run()
    states = s.output()
    want = torch.from_numpy(s.hidden()).cuda()
    assert states.shape == (46, 96) == tuple(want.shape)
    new = lambda *z, t=torch.int8: torch.zeros(*z, dtype=t, device="cuda")  # noqa: E731
    c, k, cw, kw = new(46, 96), new(46, t=torch.float32), new(46, 96), new(46, t=torch.float32)
    at = torch.cuda.current_stream().cuda_stream
    for stream in (None, at):
        c.zero_()
        torch.cuda.synchronize()
        context.quantize_tokens(states, c, k, stream=stream)
        context.quantize_tokens(want, cw, kw, stream=at)
        torch.cuda.synchronize()
        assert torch.equal(c, cw) and torch.equal(k, kw) and (k > 0).all()
    # Attention of three tokens a row to its states, which are keys and values.
    k3 = T.DeviceArray(states.buffer, (46, 3, 32), S.TURBO_DTYPE_F32)
    plan = context.cross_plan([3, 3, 3], lens, 3, 3, 32, torch.float32)
    q = torch.randn(9, 3, 32, device="cuda")
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    ws = torch.empty(max(1, plan.workspace_bytes), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    plan.run(q, k3, k3, a, workspace=ws)
    plan.run(q, want.view(46, 3, 32), want.view(46, 3, 32), b, workspace=ws)
    assert torch.equal(a, b) and (a != 0).any()
    plan.close()
    # Rows that are written and have not run are not the output's.
    s.write_tokens(ids, mask)
    assert s.output().shape == (46, 96)
    s.close()
    with pytest.raises(ValueError, match="closed"):
        context.quantize_tokens(states, c, k)
    with pytest.raises(ValueError, match="closed"):
        s.output()
    model.close()
