"""cvmk_sample (csrc/kernels/sample.cu) against its definition, whole numbers throughout."""
import numpy as np
import pytest

import operator_refs as ref

pytestmark = pytest.mark.gpu

ONE = 1 << 30
EXP = np.round((1 << 23) * np.exp(-np.arange(4096) / 256)).astype(np.int32)


@pytest.fixture(scope="module")
def kn(pkg):
    return pkg.kernels


def run(kn, x, table, scale, random, top_k=None, top_p=None, min_p=None, pad=0, skew=0, stream=None, check=True):
    """Draws from the rows of x (placed `skew` elements into an allocation, `pad` elements between rows) and compares."""
    import torch
    rows, vocab = x.shape
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    at = lambda t: 0 if t is None else t.data_ptr()
    store = np.full(skew + rows * (vocab + pad), 2**31 - 1, np.int32)   # (what lies between rows would win)
    for r in range(rows):
        store[skew + r * (vocab + pad):][:vocab] = x[r]
    store = dev(store)
    ops = [dev(np.broadcast_to(a, rows) if a is not None else None) for a in (scale, random, top_k, top_p, min_p)]
    tab = dev(table)
    token, weight, kept = (torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda") for _ in range(3))
    mass = torch.full((rows + 1,), -7, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    call = kn.Sample(logits=store.data_ptr() + 4 * skew, rows=rows, vocab=vocab, pitch=vocab + pad, table=at(tab), table_len=len(table), scale=at(ops[0]),
                     random=at(ops[1]), top_k=at(ops[2]), top_p=at(ops[3]), min_p=at(ops[4]), token=at(token), weight=at(weight), mass=at(mass), kept=at(kept))
    call.launch(stream if stream is not None else torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = [t.cpu().numpy() for t in (token, weight, mass, kept)]
    assert all(g[rows] == -7 for g in got)
    if check:
        pick = lambda a, r, off: off if a is None else int(np.broadcast_to(a, rows)[r])
        for r in range(rows):
            want = ref.sample_row(x[r], table, pick(scale, r, 0), pick(top_k, r, 0), pick(top_p, r, ONE), pick(min_p, r, 0), pick(random, r, 0))
            assert tuple(int(g[r]) for g in got) == want, (r, want)
    return got


def logits(rng, rows, vocab, kind):
    if kind == "normal":
        return np.round(rng.randn(rows, vocab) * 1500).astype(np.int32)
    if kind == "equal":
        return np.full((rows, vocab), rng.randint(-5, 5), np.int32)
    if kind == "ties":
        return rng.randint(-3, 4, (rows, vocab)).astype(np.int32) * 700
    if kind == "wide":
        return rng.randint(-2**31, 2**31, (rows, vocab), dtype=np.int64).astype(np.int32)
    x = np.full((rows, vocab), -2**31, np.int32)      # "one": a single large score
    x[np.arange(rows), rng.randint(0, vocab, rows)] = 2**31 - 1
    return x


def settings(rng, rows):
    return dict(top_k=rng.choice([-1, 0, 1, 2, 7, 50, 1000, 2**31 - 1], rows), top_p=rng.choice([-9, 0, 1, ONE // 10, ONE // 2, ONE * 9 // 10, ONE - 1, ONE, 2**31 - 1], rows),
                min_p=rng.choice([-1, 0, 1, ONE // 50, ONE // 3, ONE, 2**31 - 1], rows))


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 31, 32, 33, 100, 1000, 1025, 2047, 4099, 20011])
@pytest.mark.parametrize("kind", ["normal", "equal", "ties", "wide", "one"])
def test_rows(kn, vocab, kind):
    rng = np.random.RandomState(vocab)
    rows = 23
    x = logits(rng, rows, vocab, kind)
    scale = rng.choice([0, 1, 1000, 32768, 65536, 2**31 - 1, -4], rows) if kind != "normal" else rng.randint(20000, 60000, rows)
    random = rng.choice([0, 1, 2**30, 2**31 - 1, -1, 123456789], rows)
    for k in (0, 1):
        run(kn, x, EXP, scale, random, **(settings(rng, rows) if k else {}), pad=vocab % 3, skew=vocab % 4)


@pytest.mark.parametrize("rows", [1, 2, 9, 40, 150, 400])
def test_counts_of_rows(kn, rows):
    """From a cluster of CTAs a row to a CTA a row."""
    rng = np.random.RandomState(rows)
    run(kn, logits(rng, rows, 3001, "normal"), EXP, rng.randint(10000, 60000, rows), rng.randint(0, 2**31, rows), **settings(rng, rows))


@pytest.mark.parametrize("rows,vocab", [(1, 327680), (2, 300000), (2, 131072), (1, 50021), (30, 32000), (160, 70003), (40, 300000), (80, 150001)])
def test_large_vocabularies(kn, rows, vocab):
    rng = np.random.RandomState(vocab)
    few = min(rows, 6)   # (the definition in Python takes a second a row: the rows behind are the first ones again)
    x = logits(rng, few, vocab, "normal")
    s = settings(rng, few)
    again = np.arange(rows) % few
    got = run(kn, x[again], EXP, 30000, 987654321, **{n: v[again] for n, v in s.items()}, check=False)
    for r in range(few):
        want = ref.sample_row(x[r], EXP, 30000, int(s["top_k"][r]), int(s["top_p"][r]), int(s["min_p"][r]), 987654321)
        for i in range(r, rows, few):
            assert tuple(int(g[i]) for g in got) == want


# So many rows that slices are not kept in shared memory, at every place of a row against 16 bytes
@pytest.mark.parametrize("skew", [0, 1, 2, 3])
@pytest.mark.parametrize("filters", [False, True])
def test_many_rows(kn, skew, filters):
    rng = np.random.RandomState(skew)
    few, rows, vocab = 5, 300, 20009
    x = logits(rng, few, vocab, "normal")
    s = settings(rng, few) if filters else dict(top_k=np.zeros(few), top_p=np.full(few, ONE), min_p=np.zeros(few))
    scale, u, again = rng.randint(10000, 90000, few), rng.randint(0, 2**31, few), np.arange(rows) % few
    given = {n: v[again] for n, v in s.items()} if filters else {}
    got = run(kn, x[again], EXP, scale[again], u[again], **given, pad=skew, skew=skew, check=False)
    for r in range(few):
        want = ref.sample_row(x[r], EXP, int(scale[r]), int(s["top_k"][r]), int(s["top_p"][r]), int(s["min_p"][r]), int(u[r]))
        for i in range(r, rows, few):
            assert tuple(int(g[i]) for g in got) == want


@pytest.mark.parametrize("table", ["one", "zero", "zero_front", "rising", "negative", "long", "heavy", "steps"])
def test_tables(kn, table):
    rng = np.random.RandomState(7)
    t = {"one": [5], "zero": [0, 0, 0], "zero_front": [0, 0, 4, 3, 0], "rising": np.arange(200), "negative": [9, -3, 5, -2**31, 1],
         "long": np.round(2e9 * np.exp(-np.arange(10000) / 700)), "heavy": np.full(100, 2**31 - 1), "steps": np.repeat([4000, 3, 0, 1], 40)}[table]
    t = np.array(t, np.int64).astype(np.int32)
    for vocab, rows in ((700, 30), (9001, 10)):
        x = logits(rng, rows, vocab, "normal")
        for k in (0, 1):
            run(kn, x, t, rng.choice([0, 100, 5000, 65536], rows), rng.randint(0, 2**31, rows), **(settings(rng, rows) if k else {}))


def test_each_filter_alone_and_greedy(kn):
    rng = np.random.RandomState(3)
    x = logits(rng, 40, 5000, "ties")
    u = rng.randint(0, 2**31, 40)
    s = settings(rng, 40)
    for name, v in s.items():
        run(kn, x, EXP, 40000, u, **{name: v})
    token = run(kn, x, EXP, 40000, u, top_k=1)[0][:40]
    assert np.array_equal(token, x.argmax(1))          # the lowest index of equal scores


# Counts around what a list holds (512 elements), cuts among equal scores, weights of 31 bits
@pytest.mark.parametrize("kind", ["normal", "ties", "equal"])
@pytest.mark.parametrize("vocab", [601, 9001])
def test_long_lists(kn, vocab, kind):
    rng = np.random.RandomState(vocab + 1)
    k = np.array([33, 64, 255, 256, 257, 400, 496, 511, 512, 513, 600], np.int64)
    x = logits(rng, len(k), vocab, kind)
    u = rng.randint(0, 2**31, len(k))
    for table in (EXP, np.full(700, 2**31 - 1, np.int32), np.zeros(5, np.int32)):
        run(kn, x, table, 20000, u, top_k=k)
        run(kn, x, table, 20000, u, top_k=k, top_p=rng.choice([1, ONE // 3, ONE - 1], len(k)), min_p=rng.choice([0, ONE // 100], len(k)))


def test_the_draw_follows_the_weights(kn):
    """Random numbers at even steps: every element comes up within one step of its share."""
    x = np.array([[0, -300, -600, -100000, 0, -50]], np.int32)
    n = 4096
    token = run(kn, np.repeat(x, n, 0), EXP, 65536 // 2, (np.arange(n) * (2**31 // n)).astype(np.int64), check=False)[0][:n]
    w = EXP[np.minimum(-x[0] // 2, 4095)].astype(np.float64)
    assert np.all(np.abs(np.bincount(token, minlength=6) - n * w / w.sum()) <= 1)
    assert np.all(np.diff(token) >= 0)                 # in index order


def test_captured_and_replayed(kn):
    import torch
    rng = np.random.RandomState(5)
    rows, vocab = 12, 8000
    x = torch.from_numpy(logits(rng, rows, vocab, "normal")).cuda()
    tab, scale = torch.from_numpy(EXP).cuda(), torch.full((rows,), 30000, dtype=torch.int32, device="cuda")
    k = torch.full((rows,), 40, dtype=torch.int32, device="cuda")
    u, token = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    call = kn.Sample(logits=x.data_ptr(), rows=rows, vocab=vocab, table=tab.data_ptr(), table_len=4096, scale=scale.data_ptr(), top_k=k.data_ptr(),
                     random=u.data_ptr(), token=token.data_ptr())
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    call.launch(stream.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        call.launch(stream.cuda_stream)
    for seed in range(3):
        x.copy_(torch.from_numpy(logits(np.random.RandomState(seed), rows, vocab, "normal")))
        u.copy_(torch.from_numpy(np.random.RandomState(seed).randint(0, 2**31, rows).astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        for r in range(rows):
            assert int(token[r]) == ref.sample_row(x[r].cpu().numpy(), EXP, 30000, 40, ONE, 0, int(u[r]))[0]


def test_two_streams_at_once(kn):
    import torch
    rng = np.random.RandomState(6)
    cases = []
    for rows, vocab in ((30, 9000), (2, 120000), (200, 30001)):
        few = min(rows, 3)
        x = logits(rng, few, vocab, "normal")[np.arange(rows) % few]
        u, s = rng.randint(0, 2**31, few)[np.arange(rows) % few], settings(rng, few)
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
        ops = [dev(x), dev(EXP), dev(np.full(rows, 30000)), dev(u)] + [dev(s[n][np.arange(rows) % few]) for n in ("top_k", "top_p", "min_p")]
        token = torch.zeros(rows, dtype=torch.int32, device="cuda")
        at = [t.data_ptr() for t in ops]
        call = kn.Sample(logits=at[0], rows=rows, vocab=vocab, table=at[1], table_len=4096, scale=at[2], random=at[3], top_k=at[4], top_p=at[5], min_p=at[6],
                         token=token.data_ptr())
        want = [ref.sample_row(x[r], EXP, 30000, *(int(s[n][r]) for n in ("top_k", "top_p", "min_p")), int(u[r]))[0] for r in range(few)]
        cases.append((call, torch.cuda.Stream(), token, want, ops))
    torch.cuda.synchronize()
    for _ in range(10):
        for call, stream, *_ in cases:
            call.launch(stream.cuda_stream)
    torch.cuda.synchronize()
    for _, _, token, want, _ in cases:
        got = token.cpu().numpy()
        assert all(got[i] == want[i % len(want)] for i in range(len(got)))


def test_scores_written_by_the_kernel_before(kn, pkg):
    """dense to int32 scores, and the draw behind it on the same stream, again and again."""
    import torch
    import ctypes as ct
    rng = np.random.RandomState(8)
    lib, rows, vocab = pkg.runtime.lib(), 16, 6000
    a, b = (torch.from_numpy(np.round(rng.randn(rows, vocab) * 1500).astype(np.int32)).cuda() for _ in range(2))
    x = torch.empty_like(a)
    tab, scale, u = torch.from_numpy(EXP).cuda(), torch.full((rows,), 30000, dtype=torch.int32, device="cuda"), torch.from_numpy(rng.randint(0, 2**31, rows).astype(np.int32)).cuda()
    token = torch.zeros(rows, dtype=torch.int32, device="cuda")
    call = kn.Sample(logits=x.data_ptr(), rows=rows, vocab=vocab, table=tab.data_ptr(), table_len=4096, scale=scale.data_ptr(), random=u.data_ptr(), token=token.data_ptr())
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for turn in range(6):
        source = (a, b)[turn % 2]
        assert lib.cvmk_elemwise(ct.c_void_p(source.data_ptr()), 4, ct.c_void_p(x.data_ptr()), 4, ct.c_int64(rows * vocab), None, ct.c_void_p(stream.cuda_stream)) == 0
        call.launch(stream.cuda_stream)
        stream.synchronize()
        host = source.cpu().numpy()
        assert [int(t) for t in token] == [ref.sample_row(host[r], EXP, 30000, 0, ONE, 0, int(u[r]))[0] for r in range(rows)]
