"""Plain definitions of cvmk_dense_lut_* and cvmk_sample in whole numbers (numpy int64, Python integers), for tests."""
import numpy as np


def wrap(a):
    """int32 arithmetic: the low 32 bits as a signed number."""
    return ((np.asarray(a, np.int64) + (1 << 31)) & 0xffffffff) - (1 << 31)


def right_shift(a, by, precision):
    """cvm_right_shift for precision + by < 32."""
    top = (1 << (precision - 1)) - 1
    return np.clip(((a >> (by - 1)) + 1) >> 1, -top, top)


def chain(kn, steps, a, tensors):
    """`steps` as kernels.Chain takes them; `tensors`: address -> array of an operand."""
    for op, *v in steps:
        if op == kn.ADD_C:
            a = wrap(a + tensors[v[0]][None, :])
        elif op == kn.RSHIFT:
            a = right_shift(a, v[0], v[1])
        elif op == kn.CLIP:
            a = np.clip(a, v[0], v[1])
        elif op == kn.ADD_S:
            a = wrap(a + v[0])
        elif op == kn.MUL_S:
            a = wrap(a * v[0])
        elif op == kn.RELU:
            a = np.maximum(a, 0)
        elif op == kn.ABS:
            a = wrap(np.abs(a))
        elif op == kn.ADD_T:
            a = wrap(a + tensors[v[0]])
        elif op == kn.SUB_T:
            a = wrap(a - tensors[v[0]])
        elif op == kn.RSUB_T:
            a = wrap(tensors[v[0]] - a)
        else:
            raise AssertionError(op)
    return a


def dense_lut(kn, x, w, v, table, chain_w, chain_v, chain_y, tensors, y_dtype):
    def sums(m):   # (float64: products below 2^14, fewer than 2^17 of them, so every partial sum is a whole number below 2^31)
        return wrap(np.rint(x.astype(np.float64) @ m.astype(np.float64).T).astype(np.int64))
    a = np.clip(chain(kn, chain_w, sums(w), tensors), 0, len(table) - 1)
    t = table.astype(np.int64)[a]
    if v is not None:
        t = wrap(t * chain(kn, chain_v, sums(v), tensors))
    t = chain(kn, chain_y, t, tensors)
    return t.astype(np.int32).astype(np.int8) if y_dtype == kn.I8 else t.astype(np.int32)


def sample_row(x, table, scale, top_k, top_p, min_p, random):
    """(token, weight, mass, kept) of one row."""
    x = [int(a) for a in x]
    m, scale, one = max(x), max(int(scale), 0), 1 << 30
    w = [max(int(table[min(((m - a) * scale) >> 16, len(table) - 1)]), 0) for a in x]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    left = order[:top_k] if top_k >= 1 else order
    left = [i for i in left if w[i] << 30 >= min(max(int(min_p), 0), one) * max(int(table[0]), 0)]
    p = min(max(int(top_p), 0), one)
    if p < one:
        total, before, kept = sum(w[i] for i in left), 0, []
        for i in left:
            if before << 30 < p * total or before == 0:
                kept.append(i)
            before += w[i]
        left = kept
    mass = sum(w[i] for i in left)
    t, run, token = (int(random) & 0x7fffffff) * mass >> 31, 0, order[0]
    for i in sorted(left):
        run += w[i]
        if run > t:
            token = i
            break
    return token, w[token], mass, sum(w[i] > 0 for i in left)
