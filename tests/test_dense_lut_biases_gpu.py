"""cvmk_dense_lut_* with biases so near the ends of 32 bits that sum + bias wraps where sum + bias + rounding addend + offset does
not: columns that all lie there, and such columns among ordinary ones."""
import numpy as np
import pytest

import operator_refs as ref

pytestmark = pytest.mark.gpu

LOW, HIGH = -2**31, 2**31 - 1


@pytest.fixture(scope="module")
def kn(pkg):
    return pkg.kernels


def check(kn, rows, units, k, chain_w, chain_v, bias_w, bias_v, y_dtype, pair, extreme=False):
    """chain_w, chain_v: what follows the bias (chain_v None: not gated).  extreme: operands that are the largest a row or a unit through."""
    import torch
    rng = np.random.RandomState(rows + k)
    x, w, v = (rng.randint(-128, 128, (n, k)).astype(np.int8) for n in (rows, units, units))
    if extreme:
        x, w, v = (np.repeat(rng.choice([-128, 127], (n, 1)), k, 1).astype(np.int8) for n in (rows, units, units))
    table = rng.permutation(256).astype(np.int32) - 100
    dev = lambda a: torch.from_numpy(a).cuda()
    dx, dw, dv, dt, bw, bv = keep = [dev(a) for a in (x, w, v, table, bias_w.astype(np.int32), bias_v.astype(np.int32))]
    y = torch.full((rows, units), 77, dtype=torch.int8 if y_dtype == kn.I8 else torch.int32, device="cuda")
    at = [t.data_ptr() for t in keep]
    chains = dict(chain_w=[(kn.ADD_C, at[4])] + chain_w, chain_v=[(kn.ADD_C, at[5])] + chain_v if chain_v else [], chain_y=[])
    torch.cuda.synchronize()
    call = kn.DenseLut(x=at[0], w=at[1], v=at[2] if chain_v else 0, table=at[3], y=y.data_ptr(), rows=rows, units=units, k=k, table_len=256, table_dtype=kn.I32,
                       y_dtype=y_dtype, **chains)
    assert call.plan.kernel == pair
    call.launch(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = ref.dense_lut(kn, x, w, v if chain_v else None, table, chains["chain_w"], chains["chain_v"], [], {at[4]: bias_w, at[5]: bias_v}, y_dtype)
    assert np.array_equal(y.cpu().numpy(), want)


def near_sum(k):
    """What a sum of k products is about."""
    return int(5500 * k ** 0.5)


def biases(rng, units, low, high, mixed):
    b = rng.randint(low, high, units, dtype=np.int64)
    if mixed:
        b[rng.rand(units) < 0.5] = 1000
    return b


SHAPES = [(3, 70, 0), (40, 200, 0), (2000, 2048, 1), (2100, 1999, 1)]   # rows, units, whether on pairs of CTAs


# (shift, offset) in front of a table of 256: the addend 2^(shift - 1) + offset * 2^shift is of the size of the largest sum, K * 2^14
@pytest.mark.parametrize("rows,units,pair", SHAPES)
@pytest.mark.parametrize("k,shift,offset", [(64, 13, 128), (64, 13, -100), (16, 20, 0), (16, 12, -127)])
@pytest.mark.parametrize("mixed", [False, True])
def test_in_front_of_the_table(kn, rows, units, pair, k, shift, offset, mixed):
    rng = np.random.RandomState(shift)
    add = (1 << (shift - 1)) + offset * (1 << shift)
    ends = [(LOW, LOW + near_sum(k)), (LOW, LOW + add)] if add > 0 else [(HIGH - near_sum(k), HIGH), (HIGH + add, HIGH)]
    zero = np.zeros(units, np.int64)
    chain = [(kn.RSHIFT, shift, 8), (kn.ADD_S, offset)]
    for low, high in ends:
        for y_dtype in (kn.I8, kn.I32):
            check(kn, rows, units, k, chain, None, biases(rng, units, low, high, mixed), zero, y_dtype, pair)
            check(kn, rows, units, k, chain, [(kn.RSHIFT, 9, 8)], biases(rng, units, low, high, mixed), zero, y_dtype, pair)


# the other side, whose addend is the rounding's alone; and both sides at once
@pytest.mark.parametrize("rows,units,pair", SHAPES)
@pytest.mark.parametrize("k,shift", [(64, 22), (16, 20), (16, 23)])
@pytest.mark.parametrize("mixed", [False, True])
def test_on_the_other_side(kn, rows, units, pair, k, shift, mixed):
    rng = np.random.RandomState(shift + 1)
    assert 1 << (shift - 1) > k << 14
    far = biases(rng, units, LOW, LOW + near_sum(k), mixed)
    gate = [(kn.RSHIFT, 13, 8), (kn.ADD_S, 128)]
    near = rng.randint(-9000, 9000, units, dtype=np.int64)
    for y_dtype in (kn.I8, kn.I32):
        check(kn, rows, units, k, gate, [(kn.RSHIFT, shift, 8)], near, far, y_dtype, pair)
        check(kn, rows, units, k, gate, [(kn.RSHIFT, shift, 8)], biases(rng, units, LOW, LOW + near_sum(k), mixed), far, y_dtype, pair)


@pytest.mark.parametrize("rows,units,pair", SHAPES)
@pytest.mark.parametrize("shift,offset", [(10, 128), (9, -100), (14, 3)])
def test_largest_sums(kn, rows, units, pair, shift, offset):
    rng = np.random.RandomState(shift + 2)
    zero = np.zeros(units, np.int64)
    for low, high in ((LOW, LOW + (16 << 14)), (HIGH - (16 << 14), HIGH)):
        for mixed in (False, True):
            b = biases(rng, units, low, high, mixed)
            b[:: 7] = (LOW if low == LOW else HIGH) + (131000 if low == LOW else -131000)
            for side in (None, [(kn.RSHIFT, 9, 8)]):
                check(kn, rows, units, 16, [(kn.RSHIFT, shift, 8), (kn.ADD_S, offset)], side, b, zero, kn.I32, pair, extreme=True)
