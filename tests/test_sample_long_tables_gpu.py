"""cvmk_sample with a table too long for shared memory: shares of top_p over rows whose weights add up to far more than 32 bits."""
import numpy as np
import pytest

import operator_refs as ref
from test_sample_gpu import ONE, run

pytestmark = pytest.mark.gpu

LONG = 5000   # entries; 4096 fit shared memory


@pytest.fixture(scope="module")
def kn(pkg):
    return pkg.kernels


def check(kn, x, rows, table, scale, top_p, random, top_k=None, min_p=None, **place):
    """Every row of x, again and again until there are `rows`, with settings of its own."""
    few = len(x)
    again = np.arange(rows) % few
    pick = lambda a: None if a is None else np.broadcast_to(a, few)[again]
    got = run(kn, x[again], table, pick(scale), pick(random), top_k=pick(top_k), top_p=pick(top_p), min_p=pick(min_p), check=False, **place)
    at = lambda a, r, off: off if a is None else int(np.broadcast_to(a, few)[r])
    for r in range(few):
        want = ref.sample_row(x[r], table, at(scale, r, 0), at(top_k, r, 0), at(top_p, r, ONE), at(min_p, r, 0), at(random, r, 0))
        for i in range(r, rows, few):
            assert tuple(int(g[i]) for g in got) == want, (r, i, want)


# 65537 weights of 65535 are the last whose sum is below 2^32; 80000 equal ones of a CTA; slices of a cluster's CTAs around both
@pytest.mark.parametrize("rows,vocab", [(300, 65537), (300, 65538), (300, 65545), (300, 80000), (300, 89990), (200, 294001), (40, 327680)])
@pytest.mark.parametrize("weight", [65535, 65536, 2**24 - 1, 2**31 - 1, 0x12345678])
def test_equal_scores(kn, rows, vocab, weight):
    table = np.full(LONG, 3, np.int64)
    table[0] = weight
    x = np.full((2, vocab), -17, np.int32)
    check(kn, x, rows, table.astype(np.int32), scale=0, top_p=[int(0.9 * ONE), ONE // 7], random=[2**31 - 1, 123456789])


# one score at the type's lowest value: all others share the first digit of a distance
@pytest.mark.parametrize("top_k", [None, [0, 70000, 79000]])
@pytest.mark.parametrize("rows", [2, 300])
def test_a_masked_score(kn, rows, top_k):
    rng = np.random.RandomState(11)
    x = -rng.randint(0, 4000, (3, 80000)).astype(np.int32)
    x[:, 4321] = -2**31
    table = (65535 + (rng.randint(0, 3000, LONG) << 16)).astype(np.int32)
    check(kn, x, rows, table, scale=65536, top_p=[ONE // 3, int(0.99 * ONE), ONE - 1], random=[5, 2**30, 2**31 - 1], top_k=top_k, pad=1, skew=3)


# scores spread over all of 32 bits, and heavy entries among light ones
@pytest.mark.parametrize("rows", [3, 300])
def test_many_digits(kn, rows):
    rng = np.random.RandomState(12)
    x = np.stack([rng.randint(-2**31, 2**31, 70001), np.round(rng.randn(70001) * 1e6), rng.randint(-3, 4, 70001) * 700000]).astype(np.int32)
    table = np.where(rng.rand(LONG) < 0.5, 2**31 - 1, rng.randint(0, 70000, LONG)).astype(np.int32)
    check(kn, x, rows, table, scale=[3, 100, 70], top_p=[int(0.6 * ONE), ONE // 2, int(0.95 * ONE)], random=[2**31 - 1, 1, 2**30 + 7], min_p=[0, ONE // 1000, 0], skew=1)
