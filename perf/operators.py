"""The operators of a quantised language model's token-wise part, as cases that can be timed and compared.

Two families, both on whole numbers:
  dense_lut  dense, a table look-up as activation (cvm_lut), optionally gated by a second dense, and a residual in the
             epilogue: the feed-forward block of a decoder layer
  sample     temperature, top-k, top-p and min-p over rows of int32 logits, one random number a row

`own = False` runs their definitions in elementary torch operations; `own = True` the kernels
(cvmk_dense_lut_*, cvmk_sample) through the package's binding.
"""
import importlib
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # One token through the first half of a small decoder's feed-forward block: all latency.
        {"name": "gated_1", "op": "dense_lut", "rows": 1, "k": 2048, "units": 8192, "gated": True, "residual": False, "out": 1, "table": 256, "table_type": 1},
        # A decoding batch of a larger one: a stream of weights.
        {"name": "gated_24", "op": "dense_lut", "rows": 24, "k": 4096, "units": 16384, "gated": True, "residual": False, "out": 1, "table": 4096, "table_type": 1},
        # A few prompts' tokens, ragged in every direction, activation indices of 12 bits, wide results.
        {"name": "gated_209_odd", "op": "dense_lut", "rows": 209, "k": 1037, "units": 2777, "gated": True, "residual": False, "out": 4, "table": 4096, "table_type": 4},
        # A prefill: long enough for the tensor cores' rate.
        {"name": "gated_4096", "op": "dense_lut", "rows": 4096, "k": 4096, "units": 16384, "gated": True, "residual": False, "out": 1, "table": 256, "table_type": 1},
        # The ungated block, decoding: bias, activation and residual in the epilogue.
        {"name": "lut_8", "op": "dense_lut", "rows": 8, "k": 4096, "units": 4096, "gated": False, "residual": True, "out": 1, "table": 256, "table_type": 1},
        # The same for a batch of prompts.
        {"name": "lut_6000", "op": "dense_lut", "rows": 6000, "k": 2048, "units": 8192, "gated": False, "residual": True, "out": 1, "table": 256, "table_type": 1},
        # One sequence, a small vocabulary: latency.
        {"name": "sample_1", "op": "sample", "rows": 1, "vocab": 32000, "filters": "all", "table": 4096},
        # A decoding batch, every row with settings of its own.
        {"name": "sample_32", "op": "sample", "rows": 32, "vocab": 131072, "filters": "mixed", "table": 4096},
        # An odd vocabulary in padded rows, temperature alone.
        {"name": "sample_200_odd", "op": "sample", "rows": 200, "vocab": 50021, "filters": "none", "table": 4096},
        # The largest batch and vocabulary.
        {"name": "sample_256", "op": "sample", "rows": 256, "vocab": 262144, "filters": "mixed", "table": 4096},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, evenly spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    if rng.random() < 0.6:
        gated = rng.random() < 0.6
        c = {"op": "dense_lut", "k": _log(rng, 64, 8192), "units": _log(rng, 32, 16384), "gated": gated, "residual": rng.random() < 0.5,
             "out": rng.choice([1, 1, 4]), "table": rng.choice([256, 1000, 4096]), "table_type": rng.choice([1, 1, 4])}
        if rng.random() < 0.5:
            c["k"] = (c["k"] + 63) // 64 * 64
        c["rows"] = min(_log(rng, 1, 8192), 4096 * 4096 * 16384 // (c["k"] * c["units"]))
        return c
    c = {"op": "sample", "vocab": _log(rng, 300, 262144), "filters": rng.choice(["none", "all", "mixed", "mixed"]), "table": rng.choice([512, 4096])}
    c["rows"] = min(_log(rng, 1, 512), 256 * 262144 // c["vocab"])
    return c


class _State:
    pass


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed % (1 << 62))
    return g


def _int8(g, spread, *shape):
    """Whole numbers about 0, clipped to [-127, 127], as quantised weights and activations are."""
    return torch.randn(*shape, generator=g, device="cuda").mul_(spread).round_().clamp_(-127, 127).to(torch.int8)


def _bits(c):
    """Precision that the gate is shifted to: its values, moved by 2^(bits - 1), index the table."""
    return 8 if c["table"] == 256 else 10 if c["table"] == 1000 else 12


def _inputs(case, seed):
    s, g = _State(), _gen(seed)
    s.case = dict(case)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        s.pitch = (vocab + 3) // 4 * 4
        # 512 units of a logit to a factor e; a spread of three, a few likely tokens
        x = torch.randn(rows, s.pitch, generator=g, device="cuda") * 1500
        x += torch.randn(rows, s.pitch, generator=g, device="cuda").clamp_(min=2.5).sub_(2.5) * 4000
        s.logits = x.round_().to(torch.int32)
        n, span = case["table"], 16.0
        s.table = torch.exp(-torch.arange(n, device="cuda", dtype=torch.float64) * (span / n)).mul_(1 << 23).round_().to(torch.int32)
        heat = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64) * 0.8 + 0.5
        s.scale = (65536.0 * n / span / 512 / heat).round_().to(torch.int32)
        s.random = torch.randint(0, 1 << 31, (rows,), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        s.top_k = s.top_p = s.min_p = None
        if case["filters"] != "none":
            s.top_k = torch.randint(1, 200, (rows,), generator=g, device="cuda").to(torch.int32)
            s.top_p = (torch.rand(rows, generator=g, device="cuda", dtype=torch.float64) * 0.3 + 0.69).mul_(1 << 30).to(torch.int32)
            s.min_p = (torch.rand(rows, generator=g, device="cuda", dtype=torch.float64) * 0.05).mul_(1 << 30).to(torch.int32)
            if case["filters"] == "mixed":   # a filter that is off, one row in two or three
                s.top_k[torch.rand(rows, generator=g, device="cuda") < 0.6] = 0
                s.top_p[torch.rand(rows, generator=g, device="cuda") < 0.4] = 1 << 30
                s.min_p[torch.rand(rows, generator=g, device="cuda") < 0.6] = 0
        return s
    rows, k, units = case["rows"], case["k"], case["units"]
    s.pitch = (k + 15) // 16 * 16
    s.x = _int8(g, 40.0, rows, s.pitch)
    s.w = _int8(g, 30.0, units, s.pitch)
    s.v = _int8(g, 30.0, units, s.pitch) if case["gated"] else None
    s.bias_w, s.bias_v = (torch.randn(units, generator=g, device="cuda").mul_(2000).to(torch.int32) for _ in range(2))
    bits = _bits(case)
    spread = 1200.0 * math.sqrt(k)   # of a sum
    s.shift_w = max(1, int(round(math.log2(spread * 3.5 / (1 << (bits - 1))))))
    s.shift_v = max(1, int(round(math.log2(spread * 3.5 / 128))))
    s.offset = 1 << (bits - 1)
    # x * sigmoid(x) over [-6, 6], to 8 bits (16 where the table is wide)
    n, top = case["table"], 127 if case["table_type"] == 1 else 32767
    at = (torch.arange(n, device="cuda", dtype=torch.float64) - s.offset) * (6.0 / s.offset)
    s.table = (at * torch.sigmoid(at) * (top / 6.0)).round_().clamp_(-top, top).to(torch.int8 if case["table_type"] == 1 else torch.int32)
    s.y_shift = (7 if case["gated"] else 1) + (0 if case["table_type"] == 1 else 8)
    s.residual = _int8(g, 30.0, rows, units) if case["residual"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    K, at = importlib.import_module("cvm-runtime_b200").kernels, lambda t: 0 if t is None else t.data_ptr()
    if case["op"] == "sample":
        rows = case["rows"]
        s.token, s.weight, s.kept = (torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(3))
        s.mass = torch.empty(rows, dtype=torch.int64, device="cuda")
        s.call = K.Sample(logits=at(s.logits), rows=rows, vocab=case["vocab"], pitch=s.pitch, table=at(s.table), table_len=case["table"],
                          scale=at(s.scale), top_k=at(s.top_k), top_p=at(s.top_p), min_p=at(s.min_p), random=at(s.random),
                          token=at(s.token), weight=at(s.weight), mass=at(s.mass), kept=at(s.kept))
        return s
    s.y = torch.empty(case["rows"], case["units"], dtype=torch.int8 if case["out"] == 1 else torch.int32, device="cuda")
    s.status = torch.zeros(1, dtype=torch.int32, device="cuda")
    after = [(K.RSHIFT, s.y_shift, 8)]
    if case["residual"]:
        after += [(K.ADD_T, at(s.residual), K.I8), (K.CLIP, -127, 127)]
    s.call = K.DenseLut(x=at(s.x), x_pitch=s.pitch, w=at(s.w), v=at(s.v), w_pitch=s.pitch, rows=case["rows"], units=case["units"], k=case["k"],
                        y=at(s.y), y_dtype=case["out"], table=at(s.table), table_len=case["table"], table_dtype=case["table_type"],
                        status=at(s.status), params_static=True,
                        chain_w=[(K.ADD_C, at(s.bias_w)), (K.RSHIFT, s.shift_w, _bits(case)), (K.ADD_S, s.offset)],
                        chain_v=[(K.ADD_C, at(s.bias_v)), (K.RSHIFT, s.shift_v, 8)] if case["gated"] else [], chain_y=after)
    return s


def _shift(a, by, precision):
    """cvm_right_shift: halves round up, then a clip to the precision."""
    top = (1 << (precision - 1)) - 1
    return (((a >> (by - 1)) + 1) >> 1).clamp_(-top, top)


def _sums(x, w, k):
    """x w^T of int8 matrices: products in float32, exact over 1024 terms (1024 * 128 * 128 = 2^24)."""
    total = None
    for c in range(0, k, 1024):
        e = min(k, c + 1024)
        part = (x[:, c:e].float() @ w[:, c:e].float().t()).to(torch.int32)
        total = part if total is None else total.add_(part)
    return total


def _plain_dense(s):
    c = s.case
    a = _shift(_sums(s.x, s.w, c["k"]) + s.bias_w, s.shift_w, _bits(c)) + s.offset
    t = s.table[a.clamp_(0, c["table"] - 1).long()].int()
    if c["gated"]:
        t *= _shift(_sums(s.x, s.v, c["k"]) + s.bias_v, s.shift_v, 8)
    t = _shift(t, s.y_shift, 8)
    if s.residual is not None:
        t = (t + s.residual).clamp_(-127, 127)
    return t.to(torch.int8 if c["out"] == 1 else torch.int32)


def _plain_sample(s):
    c, one = s.case, 1 << 30
    out = []
    for r in range(0, c["rows"], 64):   # (64 rows at a time: int64 intermediates)
        part = slice(r, min(c["rows"], r + 64))
        x = s.logits[part, :c["vocab"]].long()
        ordered, order = (-x).sort(dim=1, stable=True)
        d = ordered - ordered[:, :1]
        w = s.table.long()[((d * s.scale[part, None].long()) >> 16).clamp_(max=c["table"] - 1)]
        first = w[:, :1]
        keep = torch.ones_like(w, dtype=torch.bool)
        if s.top_k is not None:
            k = s.top_k[part, None].long()
            keep &= (torch.arange(c["vocab"], device=x.device)[None] < k) | (k < 1)
            keep &= (w << 30) >= s.min_p[part, None].long().clamp(0, one) * first
            kept = torch.where(keep, w, 0)
            p, total = s.top_p[part, None].long().clamp(0, one), kept.sum(1, keepdim=True)
            need = p * (total >> 30) + ((p * (total & (one - 1)) + one - 1) >> 30)
            before = kept.cumsum(1) - kept
            keep &= (before < need) | (before == 0)
        kept = torch.where(keep, w, 0)
        mass = kept.sum(1)
        u = s.random[part].long()
        t = u * (mass >> 31) + ((u * (mass & ((1 << 31) - 1))) >> 31)
        in_place = torch.zeros_like(kept).scatter_(1, order, kept)
        token = (in_place.cumsum(1) <= t[:, None]).sum(1)
        token = torch.where(mass > 0, token, order[:, 0])
        weight = torch.zeros_like(w).scatter_(1, order, w).gather(1, token[:, None])[:, 0]
        out.append((token.int(), weight.int(), mass, (kept > 0).sum(1).int()))
    return {n: torch.cat([o[i] for o in out]) for i, n in enumerate(("token", "weight", "mass", "kept"))}


def run(s):
    if own:
        s.call.launch(torch.cuda.current_stream().cuda_stream)
        return s.y if s.case["op"] == "dense_lut" else {"token": s.token, "weight": s.weight, "mass": s.mass, "kept": s.kept}
    return _plain_dense(s) if s.case["op"] == "dense_lut" else _plain_sample(s)


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 4 + 36) + case["table"] * 4, "flops": 0}
    rows, k, units, both = case["rows"], case["k"], case["units"], 2 if case["gated"] else 1
    return {"bytes": rows * k + both * units * (k + 4) + case["table"] * case["table_type"] + rows * units * (case["out"] + (1 if case["residual"] else 0)),
            "flops": 2 * rows * k * units * both}


def _exact_dense(s):
    c = s.case

    def requantised(w, bias, by, precision):
        a = (s.x[:, :c["k"]].double() @ w[:, :c["k"]].double().t()) + bias.double()
        top = 2.0 ** (precision - 1) - 1
        return torch.floor(a / 2.0 ** by + 0.5).clamp(-top, top)   # (halves up: the same as two shifts)
    gate = (requantised(s.w, s.bias_w, s.shift_w, _bits(c)) + s.offset).clamp(0, c["table"] - 1)
    t = s.table.double()[gate.long()]
    if c["gated"]:
        t = t * requantised(s.v, s.bias_v, s.shift_v, 8)
    t = torch.floor(t / 2.0 ** s.y_shift + 0.5).clamp(-127, 127)
    if s.residual is not None:
        t = (t + s.residual.double()).clamp(-127, 127)
    return t.to(torch.int8 if c["out"] == 1 else torch.int32)


def _exact_sample(s):
    c, host = s.case, lambda t: None if t is None else t.cpu().numpy().astype(np.int64)
    logits, table, scale, random = (host(t) for t in (s.logits, s.table, s.scale, s.random))
    top_k, top_p, min_p = (host(t) for t in (s.top_k, s.top_p, s.min_p))
    rows = []
    for r in range(c["rows"]):
        x = logits[r, :c["vocab"]]
        w = table[np.minimum((x.max() - x) * scale[r] >> 16, c["table"] - 1)]
        order = np.argsort(-x, kind="stable")
        best = order[0]
        if top_k is not None:
            if top_k[r] > 0:
                order = order[:top_k[r]]
            order = order[w[order] * (1 << 30) >= min(int(min_p[r]), 1 << 30) * w[best]]
            sums = np.cumsum(w[order])
            need = -((-int(top_p[r]) * int(sums[-1])) >> 30)
            order = order[:max(1, int(np.searchsorted(sums, need)) + 1)]
        order = np.sort(order)
        sums = np.cumsum(w[order])
        mass = int(sums[-1])
        token = order[np.searchsorted(sums, (int(random[r]) * mass) >> 31, side="right")] if mass else best
        rows.append((token, w[token], mass, np.count_nonzero(w[order])))
    cols = list(zip(*rows))
    return {"token": torch.tensor(cols[0], dtype=torch.int32), "weight": torch.tensor(cols[1], dtype=torch.int32),
            "mass": torch.tensor(cols[2], dtype=torch.int64), "kept": torch.tensor(cols[3], dtype=torch.int32)}


def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_dense(s) if case["op"] == "dense_lut" else _exact_sample(s)
