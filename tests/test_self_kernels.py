"""Which kernel attention of a call's own tokens runs, without a device: the rules at their borders, and the calls that the
tests of the kernels make (test_gpu_self_kernels.py)."""
import ctypes as C

import pytest

import turboembed_amd as T
from turboembed_amd import operators as O
from turboembed_amd import seam as S
from test_operators import BF16, F16, F32, I8

CHUNKS, LOOSE, CODES, BYTES = range(4)
PROMPT, SAME, INT8 = range(3)


@pytest.mark.parametrize("call, want", [
    # Prompts: four waves share 32 rows, until blocks fill the card; F32 a wave a block of 32.
    ((23, 1, 12, 12, 64, F16), (32, 4, CHUNKS)), ((2000, 1, 12, 12, 64, BF16), (32, 4, CHUNKS)),
    ((511 * 128, 1, 1, 1, 64, BF16), (128, 4, CHUNKS)), ((511 * 128 - 1, 1, 1, 1, 64, BF16), (32, 4, CHUNKS)),
    ((511 * 128, 1, 1, 1, 64, F32), (32, 4, CHUNKS)), ((2047 * 32, 1, 1, 1, 64, F32), (32, 1, CHUNKS)),
    ((20000, 600, 1, 1, 64, F16), (128, 4, CHUNKS)), ((600, 600, 1, 1, 64, F16), (32, 4, CHUNKS)),
    ((5600, 70, 32, 8, 80, F16), (128, 4, CHUNKS)), ((5600, 70, 32, 8, 80, F32), (32, 1, CHUNKS)),
    # Rows that no chunk divides: a wave, through registers.
    ((5600, 70, 32, 8, 81, F16), (32, 1, LOOSE)), ((5600, 70, 32, 8, 64, F16, PROMPT, False), (32, 1, LOOSE)),
    # Over a cache: few rows of a sequence by 16 or 32, more by 128; F32 by 32 or 128.
    ((1, 1, 16, 4, 64, BF16, SAME), (16, 1, CHUNKS)), ((64, 64, 16, 1, 64, F16, SAME), (16, 1, CHUNKS)),
    ((64, 64, 17, 1, 64, F16, SAME), (32, 1, CHUNKS)), ((64, 64, 33, 1, 64, F16, SAME), (128, 4, CHUNKS)),
    ((1, 1, 4, 4, 64, F32, SAME), (32, 1, CHUNKS)), ((40, 1, 4, 4, 64, F32, SAME), (128, 4, CHUNKS)),
    ((40, 1, 4, 4, 63, F32, SAME), (32, 1, LOOSE)), ((40, 1, 4, 4, 64, BF16, SAME, False), (32, 1, LOOSE)),
    ((96, 96, 12, 12, 64, F16, INT8), (16, 1, BYTES)), ((96, 96, 240, 12, 64, F16, INT8), (32, 1, BYTES)),
    ((4096, 8, 32, 8, 128, BF16, INT8), (128, 4, CODES)), ((96, 96, 12, 12, 64, F32, INT8), (32, 1, CODES)),
    ((96, 96, 12, 12, 40, F16, INT8), (32, 1, CODES)), ((96, 96, 12, 12, 64, F16, INT8, False), (32, 1, CODES)),
])
def test_the_kernel_of_a_call(call, want):
    assert O.self_kernel(*call) == want


def test_what_the_hook_refuses():
    for bad in ((0, 1, 1, 1, 64, F16), (1, 0, 1, 1, 64, F16), (1, 1, 3, 2, 64, F16), (1, 1, 1, 1, 129, F16), (1, 1, 1, 1, 64, I8),
                (1, 1, 1, 1, 64, F16, 3), (1 << 30, 1, 2, 2, 64, F16), (1, 1 << 31, 1, 1, 64, F16)):
        with pytest.raises(T.TurboError):
            O.self_kernel(*bad)
    x = C.byref(C.c_uint32())
    for at in range(3):
        out = [x] * 3
        out[at] = None
        assert T.library().turbo_rocm_self_kernel(1, 1, 1, 1, 64, F16, 0, 1, *out, C.byref(S.new_error())) == S.TURBO_E_INVALID_ARGUMENT
