"""The int8 product's kernels, each of them, on an MI355X against exact sums; the tolerance is the operator's own."""
import pytest

from test_gpu_linear_i8 import TYPES, _check, _operands, _stream, _sum

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# Products that reach every kernel: which one (0: one by one, 1 to 4: pieces of so many 16 rows, 64, 128, 256: tiles),
# whether the operands are whole aligned chunks, m, n and k. Tiles with one or two stages of 128 of the inner width and
# with enough to take every buffer again, odd numbers of rows and columns among them.
KERNELS = [
    (0, False, 9, 20, 15), (0, True, 300, 257, 8),
    (1, True, 5, 700, 1024), (1, False, 16, 1003, 1537), (2, True, 2111, 17, 16), (2, False, 2059, 19, 17),
    (3, True, 4169, 17, 16), (3, False, 145, 995, 7334), (4, True, 62, 2306, 144), (4, False, 49, 2383, 16),
    (64, True, 18, 4993, 400), (64, False, 18, 4490, 390), (64, False, 5440, 19, 17),
    (128, True, 507, 7832, 272), (128, True, 1127, 3330, 400), (128, True, 4096, 1024, 768),
    (128, False, 577, 6225, 285), (128, False, 5214, 715, 400), (128, False, 7363, 3044, 4373),
    (256, True, 3330, 2835, 16), (256, True, 2369, 3607, 416), (256, True, 4794, 1666, 5760)]


@pytest.mark.parametrize("kernel, aligned, m, n, k", KERNELS)
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_every_kernel(context, kernel, aligned, m, n, k, t):
    a, a_s, w, w_s, b = _operands(m + n + k, m, n, k + (0 if aligned else 3), bias=t != "f16")
    if not aligned:
        a, w = a[:, 1:1 + k], w[:, 2:2 + k]
    wide = torch.full((m + 1, n), 7.0, dtype=TYPES[t], device="cuda")
    out = wide[:m]
    context.linear_i8(a, a_s, w, w_s, out, bias=b, stream=_stream())
    _check(out, a, a_s, w, w_s, b)
    assert (wide[m] == 7).all()
    if t != "f32":
        return
    # Exactly the sum's number, and the same for rows of the other alignment.
    one = torch.ones(max(m, n), device="cuda")
    context.linear_i8(a, one[:m], w, one[:n], out, stream=_stream())
    assert torch.equal(out, _sum(a, w).float())


@pytest.mark.parametrize("kernel, aligned, m, n, k", [c for c in KERNELS if c[0] in (3, 4, 128, 256)][::3])
def test_captured_and_replayed(context, kernel, aligned, m, n, k):
    a, a_s, w, w_s, b = _operands(5, m, n, k + (0 if aligned else 3))
    if not aligned:
        a, w = a[:, 1:1 + k], w[:, 2:2 + k]
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        context.linear_i8(a, a_s, w, w_s, out, bias=b, stream=_stream())
    for seed in range(3):
        a.copy_(_operands(seed, m, n, k)[0])
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        _check(out, a, a_s, w, w_s, b)
