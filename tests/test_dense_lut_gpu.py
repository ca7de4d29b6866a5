"""cvmk_dense_lut_* (csrc/kernels/dense_lut.cu) against its definition, bit for bit: ragged sizes, both directions of a cut
reduction, every kind of table, result and residual, streams and captured graphs."""
import numpy as np
import pytest

import operator_refs as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kn(pkg):
    return pkg.kernels


class Case:
    """Random operands of a call on the GPU, and what it has to give."""

    def __init__(self, kn, rows, k, units, gated=True, table=(256, 1), y_dtype=1, residual=None, pad=0, seed=0, low=-128, after=None, bias=True, y_pitch=None,
                 biases=9000, front=None, front_v=None):
        import torch
        rng = np.random.RandomState(seed)
        self.kn, self.rows, self.units, self.torch = kn, rows, units, torch
        pitch = (k + 15) // 16 * 16 + 16 * pad
        self.x, self.w, self.v = (rng.randint(low, 128, size=(n, pitch)).astype(np.int8) for n in (rows, units, units))
        n, kind = table
        self.table = rng.randint(-128, 128, n).astype(np.int8) if kind == 1 else rng.randint(-40000, 40000, n).astype(np.int32)
        bw, bv = (rng.randint(-biases, biases, units, dtype=np.int64).astype(np.int32) for _ in range(2))
        self.y_pitch = y_pitch or units + 3 * pad
        res = None
        if residual:
            res = rng.randint(-100, 100, size=(rows, self.y_pitch)).astype(np.int8 if residual[1] == 1 else np.int32)
        dev = lambda a: torch.from_numpy(a).cuda()
        self.keep = [dev(a) for a in (self.x, self.w, self.v, self.table, bw, bv)] + ([dev(res)] if residual else [])
        at = [t.data_ptr() for t in self.keep]
        self.y = torch.full((rows + 2, self.y_pitch), 77, dtype=torch.int8 if y_dtype == 1 else torch.int32, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        spread = 74 * 74 * np.sqrt(k)
        bits = max(2, int(np.ceil(np.log2(n))))
        sw, sv = max(1, int(np.log2(spread * 3 / 2 ** (bits - 1)))), max(1, int(np.log2(spread * 3 / 128)))
        chain_w = ([(kn.ADD_C, at[4])] if bias else []) + [(kn.RSHIFT, sw, bits), (kn.ADD_S, n // 2)]
        chain_v = ([(kn.ADD_C, at[5])] if bias else []) + [(kn.RSHIFT, sv, 8)] if gated else []
        chain_w, chain_v = chain_w if front is None else front, chain_v if front_v is None else front_v
        chain_y = [(kn.RSHIFT, (7 if gated else 1) + (0 if kind == 1 else 8), 8)] if after is None else after
        tensors = {at[4]: bw.astype(np.int64), at[5]: bv.astype(np.int64)}
        if residual:
            chain_y = chain_y + [(residual[0], at[6], residual[1])] + ([(kn.CLIP, -127, 127)] if y_dtype == 1 else [])
            tensors[at[6]] = res[:, :units].astype(np.int64)
        self.want = ref.dense_lut(kn, self.x[:, :k], self.w[:, :k], self.v[:, :k] if gated else None, self.table, chain_w, chain_v, chain_y, tensors, y_dtype)
        self.args = dict(x=at[0], w=at[1], v=at[2] if gated else 0, table=at[3], y=self.y.data_ptr(), rows=rows, units=units, k=k, table_len=n,
                         table_dtype=kind, x_pitch=pitch, w_pitch=pitch, y_pitch=self.y_pitch, y_dtype=y_dtype, chain_w=chain_w, chain_v=chain_v,
                         chain_y=chain_y, status=self.status.data_ptr())
        torch.cuda.synchronize()

    def plan(self, **change):
        return self.kn.DenseLut(**dict(self.args, **change))

    def check(self):
        self.torch.cuda.synchronize()
        got = self.y.cpu().numpy()
        assert int(self.status) == 0
        assert np.array_equal(got[:self.rows, :self.units], self.want)
        assert (got[self.rows:] == 77).all() and (got[:, self.units:] == 77).all()   # nothing else is written

    def run(self, **change):
        plan = self.plan(**change)
        plan.launch(self.torch.cuda.current_stream().cuda_stream)
        self.check()
        return plan.plan


SIZES = [(1, 16, 1), (1, 1, 1), (1, 2048, 512), (2, 5, 3), (3, 17, 65), (15, 128, 64), (16, 129, 63), (17, 300, 128), (33, 4096, 130), (48, 640, 1000),
         (64, 255, 127), (65, 64, 200), (100, 1024, 96), (128, 256, 333), (129, 512, 64), (200, 1037, 130), (255, 77, 250), (256, 512, 129),
         (257, 384, 300), (300, 1500, 257), (513, 640, 777), (1000, 96, 1031), (1030, 2050, 520)]


@pytest.mark.parametrize("rows,k,units", SIZES)
@pytest.mark.parametrize("gated", [True, False])
def test_sizes(kn, rows, k, units, gated):
    Case(kn, rows, k, units, gated, pad=rows % 2, seed=rows + k, residual=(kn.ADD_T, 1) if units % 2 else None).run(params_static=bool(k % 2))


@pytest.mark.parametrize("y_dtype", [1, 4])
def test_tiles_of_48_and_96_rows(kn, y_dtype):
    tiles = set()
    for rows, k, units in ((33, 3051, 10231), (209, 1037, 2777), (517, 3340, 193), (2985, 5312, 84), (3904, 2368, 130)):
        plan = Case(kn, rows, k, units, units < 10000, (256, 1), y_dtype, seed=rows, pad=1).run()
        tiles.add(plan.row_tile)
    assert {48, 96} <= tiles


@pytest.mark.parametrize("rows,k,units", [(1, 256, 70), (37, 300, 200), (260, 192, 150), (700, 130, 300)])
@pytest.mark.parametrize("table", [(1, 1), (2, 4), (300, 1), (1000, 4), (4096, 4), (4097, 4), (20000, 1)])
@pytest.mark.parametrize("y_dtype", [1, 4])
def test_tables_and_results(kn, rows, k, units, table, y_dtype):
    for gated in (True, False):
        Case(kn, rows, k, units, gated, table, y_dtype, seed=table[0], pad=1, bias=table[0] % 2 == 0).run()


@pytest.mark.parametrize("rows,units", [(5, 48), (40, 97), (300, 160)])
@pytest.mark.parametrize("step", ["ADD_T", "SUB_T", "RSUB_T"])
@pytest.mark.parametrize("kind", [1, 4])
def test_residuals(kn, rows, units, step, kind):
    for y_dtype in (1, 4):
        for pad in (0, 1):
            Case(kn, rows, 144, units, rows % 2 == 0, (256, 1), y_dtype, (getattr(kn, step), kind), pad, seed=units).run()


def test_steps_that_are_rare(kn):
    """Chains of many steps, products that wrap, results whose low byte is stored."""
    for rows in (9, 270):
        Case(kn, rows, 512, 100, True, (256, 4), 1, after=[(kn.MUL_S, 1 << 20), (kn.ABS,), (kn.ADD_S, -5), (kn.RELU,)], seed=3).run()
        Case(kn, rows, 512, 100, True, (256, 4), 4, after=[], seed=4).run()


def test_largest_reduction(kn):
    c = Case(kn, 2, (1 << 17) - 1, 3, True, (256, 1), 4, seed=1)
    c.run()
    full = Case(kn, 1, (1 << 17) - 1, 2, False, (4096, 4), 4, seed=1, low=127)   # every sum is 127 * 127 * K
    full.run()


def test_weights_written_by_the_kernel_before(kn, pkg):
    """params_static = 0: weights, bias and table that a kernel of the same stream still writes when this one may start."""
    import torch
    import kernel_desc as kd
    import ctypes as ct
    lib = pkg.runtime.lib()
    c = Case(kn, 4, 512, 192, seed=9)
    words = [t.view(torch.int32).reshape(-1) for t in c.keep[1:6]]
    params = torch.cat(words)
    rows = 50000
    source = torch.zeros(rows, params.numel(), dtype=torch.int32, device="cuda") if params.numel() < 20000 else None
    rows = rows if source is not None else 4000
    source = torch.zeros(rows, params.numel(), dtype=torch.int32, device="cuda")
    source[-1] = params
    target = torch.zeros_like(params)
    at, args = target.data_ptr(), {}
    offsets = np.cumsum([0] + [t.numel() * 4 for t in words])
    for name, o in zip(("w", "v", "table"), offsets):
        args[name] = at + int(o)
    args["chain_w"] = [(kn.ADD_C, at + int(offsets[3]))] + c.args["chain_w"][1:]
    args["chain_v"] = [(kn.ADD_C, at + int(offsets[4]))] + c.args["chain_v"][1:]
    plan = c.plan(**args)
    total = kd.Reduce(n_keep=1, n_red=1, x=source.data_ptr(), x_dtype=4, y=at, y_dtype=4)
    total.keep_extent[0], total.keep_stride[0], total.red_extent[0], total.red_stride[0] = params.numel(), 1, rows, params.numel()
    stream = torch.cuda.Stream()
    for _ in range(2):
        target.zero_()
        torch.cuda.synchronize()
        assert lib.cvmk_reduce(ct.byref(total), ct.c_void_p(stream.cuda_stream)) == 0
        plan.launch(stream.cuda_stream)
        c.check()


def test_a_chain_of_launches_and_a_graph(kn):
    """A result that is the next launch's input, eagerly and replayed from a graph with other inputs; no synchronisation in between."""
    import torch
    for rows in (3, 290):
        a = Case(kn, rows, 256, 320, seed=21)
        b = Case(kn, rows, 320, 128, seed=22)
        first = a.plan(y_pitch=320)
        second = b.plan(x=a.y.data_ptr(), x_pitch=320)
        stream = torch.cuda.Stream()

        def want():
            middle = ref.dense_lut(kn, a.x[:, :256], a.w[:, :256], a.v[:, :256], a.table, a.args["chain_w"], a.args["chain_v"], a.args["chain_y"],
                                   {t.data_ptr(): t.cpu().numpy().astype(np.int64) for t in a.keep[4:6]}, 1)
            return ref.dense_lut(kn, middle, b.w[:, :320], b.v[:, :320], b.table, b.args["chain_w"], b.args["chain_v"], b.args["chain_y"],
                                 {t.data_ptr(): t.cpu().numpy().astype(np.int64) for t in b.keep[4:6]}, 1)
        for _ in range(3):
            first.launch(stream.cuda_stream)
            second.launch(stream.cuda_stream)
        b.want = want()
        b.check()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            first.launch(stream.cuda_stream)
            second.launch(stream.cuda_stream)
        a.x = a.x[::-1].copy()
        a.keep[0].copy_(torch.from_numpy(a.x))
        b.y.fill_(77)
        graph.replay()
        graph.replay()
        b.want = want()
        b.check()


def test_two_streams_at_once(kn):
    import torch
    a, b = Case(kn, 20, 2048, 2000, seed=31), Case(kn, 400, 512, 900, False, seed=32)
    plans = [(a.plan(), torch.cuda.Stream()), (b.plan(), torch.cuda.Stream())]
    for _ in range(20):
        for plan, stream in plans:
            plan.launch(stream.cuda_stream)
    a.check()
    b.check()


def test_a_plan_of_another_device_is_refused(kn):
    case = Case(kn, 5, 256, 300, seed=33)
    plan = case.plan()
    plan.plan.device += 1
    with pytest.raises(kn.KernelError) as refused:
        plan.launch()
    assert refused.value.status == kn.ERR_ARG
    plan.plan.device -= 1
    plan.launch()
    case.check()


def test_a_residual_that_is_the_result(kn):
    """y += ...: the tensor operand may be y itself."""
    import torch
    for rows in (6, 300):
        c = Case(kn, rows, 160, 90, False, residual=(kn.ADD_T, 1), seed=5)
        c.y[:rows].copy_(c.keep[6])
        res = c.keep[6].cpu().numpy()
        c.plan(chain_y=[s if s[0] != kn.ADD_T else (kn.ADD_T, c.y.data_ptr(), 1) for s in c.args["chain_y"]]).launch(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert np.array_equal(c.y.cpu().numpy()[:rows], c.want) and res.shape == c.want.shape


# Rows of y on 16 bytes that are longer than the result: nothing behind the units is touched
@pytest.mark.parametrize("rows,units,pitch", [(5, 100, 112), (300, 100, 112), (300, 257, 288), (2100, 33, 48), (700, 1000, 1008)])
@pytest.mark.parametrize("y_dtype", [1, 4])
@pytest.mark.parametrize("residual", [None, 1, 4])
def test_rows_longer_than_the_result(kn, rows, units, pitch, y_dtype, residual):
    for gated in (True, False):
        for table in ((256, 1), (300, 4)):
            Case(kn, rows, 1100, units, gated, table, y_dtype, (kn.ADD_T, residual) if residual else None, seed=pitch, y_pitch=pitch).run()


# Biases near the ends of 32 bits, whose sums wrap: some of a tile's, or all
@pytest.mark.parametrize("rows,units", [(3, 70), (40, 200), (1100, 1000)])
@pytest.mark.parametrize("gated", [True, False])
def test_sums_that_wrap(kn, rows, units, gated):
    for biases in (2**31 - 1, 2**31 - 2**20, 2**25):
        Case(kn, rows, 900, units, gated, biases=biases, seed=units, y_pitch=(units + 15) // 16 * 16).run()


# Chains that are not a shift (and a sum with a constant) in front of the table, or on the other side
@pytest.mark.parametrize("rows,units", [(3, 70), (1100, 1000)])
@pytest.mark.parametrize("front", range(6))
def test_other_chains(kn, rows, units, front):
    w = [[], [(kn.RELU,), (kn.RSHIFT, 12, 8)], [(kn.MUL_S, 3), (kn.RSHIFT, 14, 8), (kn.ADD_S, 128), (kn.ABS,)], [(kn.RSHIFT, 11, 8), (kn.ADD_S, -300)],
         [(kn.RSHIFT, 11, 8), (kn.ADD_S, 400)], [(kn.CLIP, -100000, 90000), (kn.RSHIFT, 9, 9), (kn.CLIP, 0, 250)]][front]
    v = [[], [(kn.CLIP, -50, 50)], [(kn.RSHIFT, 13, 8), (kn.ADD_S, 7)], [(kn.RELU,), (kn.RSHIFT, 12, 8)], [(kn.RSHIFT, 20, 8)], [(kn.RSHIFT, 1, 16)]][front]
    for gated in (True, False):
        for y_dtype, after in ((4, []), (1, None)):
            Case(kn, rows, 500, units, gated, (256, 1), y_dtype, after=after, front=w, front_v=v if gated else None, seed=front).run()


# Pairs of CTAs, results whose rows end off 16 bytes; tables that stay where they lie, and a chain step by step
@pytest.mark.parametrize("rows,k,units", [(1100, 70, 6973), (2100, 130, 1999)])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("residual", [None, ("ADD_T", 1), ("RSUB_T", 4)])
@pytest.mark.parametrize("table", [(256, 1), (1000, 4), (20000, 1)])
def test_pairs_off_16_bytes(kn, rows, k, units, gated, residual, table):
    for y_dtype in (1, 4):
        for front in (None, [(kn.CLIP, -100000, 90000), (kn.RSHIFT, 9, 9), (kn.CLIP, 0, 250)]):
            plan = Case(kn, rows, k, units, gated, table, y_dtype, (getattr(kn, residual[0]), residual[1]) if residual else None, seed=units, front=front).run()
            assert plan.kernel == 1 and plan.io == 0


def test_sizes_drawn_at_random(kn):
    """Every cut that sizes of 1 to 3000 rows, 1 to 3000 long, 1 to 3000 units lead to, and two that lead to pairs of CTAs."""
    rng = np.random.RandomState(17)
    cuts = set()
    for i in range(60):
        rows, k, units = (int(np.exp(rng.uniform(0, np.log(3000)))) for _ in range(3))
        plan = Case(kn, rows, k, units, i % 2 == 0, [(256, 1), (1000, 4)][i % 3 == 0], [1, 4][i % 5 == 0], (kn.ADD_T, 1) if i % 4 == 0 else None, seed=i,
                    y_pitch=(units + 15) // 16 * 16 if i % 7 < 3 else None).run(params_static=bool(i % 2))
        cuts.add((plan.kernel, plan.split))
    for rows, k, units in ((300, 1200, 9000), (2800, 900, 2900)):
        cuts.add((Case(kn, rows, k, units, seed=rows).run().kernel, 1))
    assert {kernel for kernel, _ in cuts} == {0, 1} and max(split for _, split in cuts) > 1


def test_whole_rows_drawn_at_random(kn):
    """Units that end on 16 bytes: results and operands that go by TMA."""
    rng = np.random.RandomState(18)
    ways = set()
    for i in range(40):
        rows, k, units = (int(np.exp(rng.uniform(np.log(lo), np.log(hi)))) for lo, hi in ((257, 3000), (1, 1000), (16, 3000)))
        units = (units + 15) // 16 * 16
        plan = Case(kn, rows, k, units, i % 2 == 0, [(256, 1), (1000, 4)][i % 3 == 0], [1, 4][i % 5 < 2], (kn.SUB_T, 1) if i % 4 < 2 else None, seed=i,
                    y_pitch=units + 16 * (i % 7 < 3)).run(params_static=bool(i % 2))
        ways.add((plan.kernel, plan.io))
    assert ways >= {(1, 1), (1, 2)}
