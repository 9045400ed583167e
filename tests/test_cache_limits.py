"""Attention over a cache: calls whose work is past what the device counts it in are refused, without a device."""
import pytest

from test_cache import CAPACITY, N, P, PAGE, _attend, _cache
from test_operators import F16, GB, I32, I8, NO_CONTEXT, Fake, _status
from turboembed_amd import operators as O


@pytest.mark.parametrize("share, tokens, columns, want", [
    (1 << 24, 64, 1 << 26, (CAPACITY, 0)),       # 2^30 rows of 2^24 heads over 2^30 positions: past 64 bits
    (1 << 30, 1, 1 << 20, (CAPACITY, 0)),
    (1 << 20, 1, 1 << 10, NO_CONTEXT),
    (128, 1 << 16, 1 << 26, NO_CONTEXT),         # 2^23 rows over 2^30 positions
    (8, 1 << 20, 1 << 20, NO_CONTEXT),
    (1, 1 << 30, 1 << 26, NO_CONTEXT),
])
def test_work_past_its_count_is_refused(share, tokens, columns, want):
    need = O.cache_workspace(tokens, N, share, 1, 8, F16)
    rows = dict(q=Fake(40 * GB, (tokens, share, 8), F16), out=Fake(80 * GB, (tokens, share, 8), F16),
                workspace=Fake(200 * GB, (need,), I8), pages=Fake(120 * GB, (N, columns), I32, (0, 1)))
    cache = _cache(k=Fake(10 * GB, (P * PAGE, 1, 8), F16), v=Fake(30 * GB, (P * PAGE, 1, 8), F16))
    assert _status(_attend, cache=cache, **rows) == want
