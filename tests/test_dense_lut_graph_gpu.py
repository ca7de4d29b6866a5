"""Feed-forward blocks of graphs (dense, cvm_lut, broadcast_mul, ...) that the executor runs in one launch, and graphs that
look like them and are not: the oracle's results, and whether the launch was made."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def steps(rt, js, pb, x):
    net = rt.CVMAPILoadModel(js, pb, 0)
    try:
        out = rt.inference_bytes(net, x).copy()
        return out, [label for label, _ in rt.profile_steps(net, x)]
    finally:
        rt.CVMAPIFreeModel(net)


def check(rt, oracle, model, fused):
    js, pb, x = model
    got, labels = steps(rt, js, pb, x)
    assert np.array_equal(got, oracle.run_model(js, pb, x))
    assert sum(label.startswith("dense_lut:") for label in labels) == fused, labels
    return labels


@pytest.mark.parametrize("rows,hidden,inner,vocab", [(1, 64, 128, 100), (3, 256, 512, 1000), (40, 128, 333, 77), (300, 96, 640, 500)])
@pytest.mark.parametrize("gated", [True, False])
def test_decoder(rt, wl, oracle, rows, hidden, inner, vocab, gated):
    check(rt, oracle, wl.decoder_mlp(rows, hidden, inner, 2, vocab, gated=gated), 2)


class Build:
    """One block over (rows, k) of data, put together by `body`."""

    def __init__(self, wl, body, rows=7, k=64, seed=3):
        g = wl.GraphBuilder(seed)
        x = g.var("data", (rows, k), 8)
        js, pb = g.finish(body(g, x))
        self.model = (js, pb, np.random.RandomState(seed).randint(-127, 128, size=(rows, k)).astype(np.int8))


def shift(g, x, by=9, precision=8):
    return g.op("cvm_right_shift", [x], g.shape_of(x), {"precision": precision, "shift_bit": by})


def clip(g, x, precision=8):
    return g.op("cvm_clip", [x], g.shape_of(x), {"precision": precision})


def table(wl, g, x, bits=8):
    return g.lut(x, wl.silu_table(bits), 8, 1 << (bits - 1))


def mul(g, a, b):
    return g.op("broadcast_mul", [a, b], g.shape_of(a))


FUSED = {
    "ungated": lambda wl, g, x: table(wl, g, g.dense(x, 48, 9)),
    "no_bias": lambda wl, g, x: table(wl, g, g.dense(x, 48, 9, bias=False)),
    "relu_in_front": lambda wl, g, x: table(wl, g, g.dense(x, 48, 9, relu=True)),
    "index_as_it_is": lambda wl, g, x: g.lut(g.dense(x, 48), np.arange(-60, 60, dtype=np.int8), 8),
    "wide_table": lambda wl, g, x: clip(g, shift(g, g.lut(g.dense(x, 48, 9), (np.arange(200) * 977).astype(np.int32), 20, 100), 5)),
    "table_of_one": lambda wl, g, x: g.lut(g.dense(x, 48, 9), np.array([5], np.int8), 8),
    "gated": lambda wl, g, x: g.gated(x, 48),
    "gate_second": lambda wl, g, x: shift(g, mul(g, g.dense(x, 48, 9), table(wl, g, g.dense(x, 48, 9))), 7),
    "operands_swapped": lambda wl, g, x: shift(g, mul(g, *[table(wl, g, g.dense(x, 40, 9)), g.dense(x, 40, 9)][::-1]), 7),
    "steps_behind_the_table": lambda wl, g, x: shift(g, mul(g, shift(g, g.lut(g.dense(x, 48, 9), (np.arange(256) * 300 - 30000).astype(np.int32), 17, 128), 9),
                                                            g.dense(x, 48, 9)), 7),
    "product_as_it_is": lambda wl, g, x: mul(g, table(wl, g, g.dense(x, 48, 9)), g.dense(x, 48, 9)),
    "sides_of_12_bits": lambda wl, g, x: shift(g, mul(g, table(wl, g, shift(g, g.dense(x, 48), 5, 12), 12), shift(g, g.dense(x, 48), 7, 10)), 9),
}


@pytest.mark.parametrize("name", FUSED)
@pytest.mark.parametrize("rows", [5, 260])
def test_blocks_in_one_launch(rt, wl, oracle, name, rows):
    check(rt, oracle, Build(wl, lambda g, x: FUSED[name](wl, g, x), rows).model, 1)


def residual(wl, g, x):
    y = table(wl, g, g.dense(x, 64, 9))
    return clip(g, g.op("elemwise_add", [y, x], g.shape_of(y)))


def subtracted(wl, g, x):
    other = g.dense(x, 48, 9)
    y = g.gated(x, 48)
    return clip(g, g.op("elemwise_sub", [other, y], g.shape_of(y)))


@pytest.mark.parametrize("body", [residual, subtracted])
@pytest.mark.parametrize("rows", [5, 260])
def test_a_sum_behind_it(rt, wl, oracle, body, rows):
    labels = check(rt, oracle, Build(wl, lambda g, x: body(wl, g, x), rows).model, 1)
    assert not any(label.startswith(("elemwise", "cvm_clip")) for label in labels)


def used_twice(wl, g, x):
    a = g.dense(x, 48, 9)
    return clip(g, g.op("elemwise_add", [table(wl, g, a), a], g.shape_of(a)))


def other_input(wl, g, x):
    z = g.dense(x, 64, 9)
    return shift(g, mul(g, table(wl, g, g.dense(x, 48, 9)), g.dense(z, 48, 9)), 7)


def computed_table_index_twice(wl, g, x):
    return shift(g, mul(g, table(wl, g, g.dense(x, 48, 9)), table(wl, g, g.dense(x, 48, 9))), 7)


@pytest.mark.parametrize("body,rows,k,fused", [(used_twice, 5, 64, 0), (other_input, 5, 64, 1), (computed_table_index_twice, 5, 64, 2),
                                               (lambda wl, g, x: g.gated(x, 48), 5, 60, 0),       # rows of 60 bytes
                                               (lambda wl, g, x: g.dense(x, 48, 9), 5, 64, 0)])
def test_what_stays_apart(rt, wl, oracle, body, rows, k, fused):
    check(rt, oracle, Build(wl, lambda g, x: body(wl, g, x), rows, k).model, fused)


def test_a_head_in_the_middle(rt, wl, oracle):
    def body(g, x):
        a = g.dense(x, 48, 9)
        return [table(wl, g, a), a]
    check(rt, oracle, Build(wl, body).model, 0)


def test_a_decoding_step(rt, wl, oracle, pkg):
    """As a server would run it: the token-wise part of a model by CVMAPIInference, scores to tokens by cvmk_sample, and the
    tokens' vectors taken from a table for the next step."""
    import torch
    import operator_refs as ref
    kn = pkg.kernels
    rows, hidden, vocab = 6, 128, 700
    js, pb, x = wl.decoder_mlp(rows, hidden, 256, 2, vocab)
    rng = np.random.RandomState(1)
    vectors = rng.randint(-127, 128, size=(vocab, hidden)).astype(np.int8)
    weights = np.round((1 << 20) * np.exp(-np.arange(2048) / 128)).astype(np.int32)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    tab, scale, top_k, top_p = dev(weights), torch.full((rows,), 40, dtype=torch.int32, device="cuda"), torch.full((rows,), 50, dtype=torch.int32, device="cuda"), \
        torch.full((rows,), int(0.9 * 2**30), dtype=torch.int32, device="cuda")
    token = torch.empty(rows, dtype=torch.int32, device="cuda")
    net = rt.CVMAPILoadModel(js, pb, 0)
    seen = set()
    try:
        for turn in range(4):
            scores = rt.inference_bytes(net, x).view(np.int32).reshape(rows, vocab)
            assert np.array_equal(scores.reshape(-1).view(np.uint8), oracle.run_model(js, pb, x))
            u = rng.randint(0, 2**31, rows).astype(np.int32)
            logits, random = dev(scores), dev(u)
            kn.Sample(logits=logits.data_ptr(), rows=rows, vocab=vocab, table=tab.data_ptr(), table_len=2048, scale=scale.data_ptr(), top_k=top_k.data_ptr(),
                      top_p=top_p.data_ptr(), random=random.data_ptr(), token=token.data_ptr()).launch(torch.cuda.current_stream().cuda_stream)
            drawn = token.cpu().numpy()
            assert [int(t) for t in drawn] == [ref.sample_row(scores[r], weights, 40, 50, int(0.9 * 2**30), 0, int(u[r]))[0] for r in range(rows)]
            seen.update(drawn.tolist())
            x = vectors[drawn]
    finally:
        rt.CVMAPIFreeModel(net)
    assert len(seen) > rows
