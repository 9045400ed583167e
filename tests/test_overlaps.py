"""What the operators take for an overlap of two arrays, without a device: K and V of a cache that lie between each other
are none, whatever step they share."""
import random

import pytest

from test_cache import _attend, _cache, _read, _write
from test_operators import ARG, F16, GB, I8, NO_CONTEXT, Fake, _status

S, K, W = 96, 2, 40     # (test_cache's slots, key heads and width)

# Strides of slots and heads, V's first element, and a place where a head of K has its last.
BETWEEN = [
    # Side by side in a slot, in a head of a slot, in a head, and in a head's plane of slots; with room between.
    ((2 * K * W, W), K * W, K * W - 1), ((K * 2 * W, 2 * W), W, W - 1), ((2 * W, S * 2 * W), W, W - 1),
    ((W, 2 * S * W), S * W, S * W - 1), ((K * 3 * W + 8, 3 * W), 2 * W, W - 1), ((K * 2 * W + 80, 2 * W), W, W - 1)]


@pytest.mark.parametrize("strides, second, taken", BETWEEN)
def test_states_between_each_other(strides, second, taken):
    for t, size in ((F16, 2), (I8, 1)):
        k, v = (Fake(10 * GB + size * at, (S, K, W), t, (*strides, 1)) for at in (0, second))
        for a, b in ((k, v), (v, k)):
            cache = _cache(t, k=a, v=b)
            assert _status(_write, cache=cache) == NO_CONTEXT           # (whose outputs they are)
            assert _status(_read, cache=cache) == NO_CONTEXT and _status(_attend, cache=cache) == NO_CONTEXT
        # ...and where they do meet.
        near = Fake(10 * GB + size * taken, (S, K, W), t, (*strides, 1))
        assert _status(_write, cache=_cache(t, k=k, v=near)) == (ARG, 4)
        assert _status(_write, cache=_cache(t, k=near, v=k)) == (ARG, 4)


def test_no_overlap_is_missed():
    """Arrays of few elements at random: whatever shares a byte is refused."""
    rng, found = random.Random(1), 0
    for _ in range(20000):
        def some(t):
            n = [rng.choice([1, 1, 2, 3, 4]) for _ in range(2)]
            return (*n, rng.choice([1, 2, 3])), (rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 24]), rng.choice([0, 1, 2, 3, 4, 6, 8, 12]), 1)

        shape, ks = some(F16)
        vs = some(F16)[1]
        at = rng.randrange(0, 24)

        def places(base, strides):
            return [base + i * strides[0] + j * strides[1] + c for i in range(shape[0]) for j in range(shape[1]) for c in range(shape[2])]
        mine, other = places(0, ks), places(at, vs)
        cache = _cache(page=1, k=Fake(10 * GB, shape, F16, ks), v=Fake(10 * GB + 2 * at, shape, F16, vs))
        rows = dict(k=Fake(GB, (5, *shape[1:]), F16), v=Fake(2 * GB, (5, *shape[1:]), F16))
        got = _status(_write, cache=cache, **rows)
        if set(mine) & set(other) or len(set(mine)) < len(mine) or len(set(other)) < len(other):
            assert got in ((ARG, 3), (ARG, 4)), (shape, ks, vs, at)
            found += 1
    assert found > 5000
