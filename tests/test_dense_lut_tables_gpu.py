"""Tables of cvmk_dense_lut_* that are copied to shared memory: lengths around what a thread copies at once, addresses off 16 bytes,
entries that go through steps on the way, and tables that a graph's executor has taken through such steps at load."""
import numpy as np
import pytest

from test_dense_lut_gpu import Case
from test_dense_lut_graph_gpu import Build, check, clip, mul, shift

pytestmark = pytest.mark.gpu

ENTRIES = [(255, 1), (256, 4), (257, 1), (511, 4), (513, 1), (1027, 4), (2049, 1), (4095, 4), (4096, 4), (4097, 1), (10000, 1), (16383, 1), (16384, 1)]


@pytest.fixture(scope="module")
def kn(pkg):
    return pkg.kernels


@pytest.mark.parametrize("table", ENTRIES)
@pytest.mark.parametrize("rows,units", [(5, 70), (1400, 2000)])
@pytest.mark.parametrize("gated", [True, False])
def test_lengths_and_places(kn, table, rows, units, gated):
    import torch
    n, kind = table
    for after in (None, [], [(kn.ADD_S, 100000), (kn.MUL_S, 3)]):
        c = Case(kn, rows, 48, units, gated, table, 4, after=after, seed=n)
        assert c.plan().plan.kernel == (rows > 1000)
        for off in (0, 1, 3):   # entries in front
            moved = torch.zeros(n + off, dtype=c.keep[3].dtype, device="cuda")
            moved[off:] = c.keep[3]
            c.y.fill_(77)
            torch.cuda.synchronize()
            c.run(table=moved.data_ptr() + off * kind, params_static=bool(off))


def scalars(g, x, pairs):
    for op, value in pairs:
        x = g.op(op, [x, g.var("s%d" % len(g.params), (1,), abs(value).bit_length() + 1, np.array([value], np.int32))], g.shape_of(x))
    return x


NARROW, WIDE = (np.arange(10000) % 251 - 125).astype(np.int8), (np.arange(4000) * 31 - 60000).astype(np.int32)
BEHIND = {
    "narrow_stays": lambda g, y: clip(g, scalars(g, y, [("broadcast_add", 5)])),
    "narrow_widens": lambda g, y: scalars(g, y, [("broadcast_mul", 300), ("broadcast_add", -7)]),
    "wide_narrows": lambda g, y: shift(g, y, 10),
    "many": lambda g, y: clip(g, scalars(g, y, [("broadcast_add", 9), ("broadcast_sub", 4), ("broadcast_max", -40), ("broadcast_add", 1), ("broadcast_mul", 2),
                                               ("broadcast_add", -3), ("broadcast_max", -50), ("broadcast_add", 2), ("broadcast_max", -45), ("broadcast_add", 3)])),
    "absolute": lambda g, y: g.op("abs", [y], g.shape_of(y)),
}


@pytest.mark.parametrize("name", BEHIND)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("rows", [5, 300])
def test_steps_behind_a_table(rt, wl, oracle, name, wide, rows):
    def table(g, x):
        t = WIDE if wide else NARROW
        y = g.lut(shift(g, g.dense(x, 48), 4, 14 if not wide else 12), t, 18 if wide else 8, len(t) // 2)
        return BEHIND[name](g, y)
    check(rt, oracle, Build(wl, table, rows).model, 1)
    check(rt, oracle, Build(wl, lambda g, x: shift(g, mul(g, shift(g, table(g, x), 6, 8), g.dense(x, 48, 9)), 7), rows).model, 1)

    def joined(g, x):
        y = clip(g, table(g, x))
        return clip(g, g.op("elemwise_add", [y, g.dense(x, 48, 9)], g.shape_of(y)))
    check(rt, oracle, Build(wl, joined, rows).model, 1)
