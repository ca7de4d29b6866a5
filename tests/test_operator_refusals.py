"""cvmk_dense_lut_* and cvmk_sample: what they refuse, and calls of nothing.  No device is needed: every refusal comes
before the first CUDA call, and addresses are never followed."""
import ctypes as ct

import pytest


@pytest.fixture(scope="module")
def kn(pkg):
    return pkg.kernels


def dense(kn, **change):
    a = dict(x=1 << 20, w=2 << 20, v=3 << 20, table=4 << 20, y=5 << 20, rows=5, units=40, k=64, table_len=256,
             chain_w=[(kn.ADD_C, 6 << 20), (kn.RSHIFT, 9, 8), (kn.ADD_S, 128)], chain_v=[(kn.RSHIFT, 9, 8)],
             chain_y=[(kn.RSHIFT, 7, 8), (kn.ADD_T, 7 << 20, kn.I8)])
    a.update(change)
    return kn.DenseLut(**a)


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "sizes"), (dict(units=0), "sizes"), (dict(k=0), "sizes"), (dict(k=1 << 17), "sizes"),
    (dict(rows=1 << 30, units=1 << 30), "too many outputs"), (dict(rows=2**31 - 1), "too many outputs"),
    (dict(y_dtype=2), "int8 or int32"), (dict(table_dtype=0), "int8 or int32"), (dict(table_len=0), "at least one entry"),
    (dict(k=65, x_pitch=80), "multiples of 16"), (dict(k=65, w_pitch=80), "multiples of 16"), (dict(x_pitch=72), "multiples of 16"),
    (dict(x_pitch=48), "shorter"), (dict(w_pitch=32), "shorter"), (dict(y_pitch=39), "shorter"), (dict(y_pitch=-1), "shorter"),
    (dict(x_pitch=1 << 40), "too far apart"),
    (dict(v=0), "chain_v without v"),
    (dict(chain_w="late_bias"), "first step"), (dict(chain_y="bias"), "first step"),
    (dict(chain_w="tensor"), "one tensor step"), (dict(chain_v="tensor"), "one tensor step"), (dict(chain_y="two"), "one tensor step"),
    (dict(chain_y="type"), "int8 or int32"), (dict(chain_w="null_bias"), "tensor operand"), (dict(chain_y="null"), "tensor operand"),
    (dict(chain_w="shift"), "bad attributes"), (dict(chain_v="unknown"), "unknown step"),
    (dict(x=0), "null operand"), (dict(w=0), "null operand"), (dict(y=0), "null operand"), (dict(table=0), "null operand"),
    (dict(x=(1 << 20) + 8), "16-byte aligned"), (dict(w=(1 << 20) + 8), "16-byte aligned"), (dict(v=(1 << 20) + 1), "16-byte aligned"),
    (dict(y=(1 << 20) + 2, y_dtype=4), "aligned to its elements"), (dict(table=(1 << 20) + 2, table_dtype=4), "aligned to its elements"),
    (dict(chain_w="odd_bias"), "aligned to its elements"), (dict(chain_y="odd"), "aligned to its elements"),
])
def test_dense_lut_refuses(kn, change, text):
    chains = {"late_bias": [(kn.RELU,), (kn.ADD_C, 1 << 20)], "bias": [(kn.ADD_C, 1 << 20)], "tensor": [(kn.ADD_T, 1 << 20, kn.I8)],
              "two": [(kn.ADD_T, 1 << 20, kn.I8), (kn.SUB_T, 1 << 20, kn.I8)], "type": [(kn.RSUB_T, 1 << 20, 2)], "null_bias": [(kn.ADD_C, 0)],
              "null": [(kn.ADD_T, 0, kn.I8)], "shift": [(kn.RSHIFT, 33, 8)], "unknown": [(77,)], "odd_bias": [(kn.ADD_C, (1 << 20) + 1)],
              "odd": [(kn.ADD_T, (1 << 20) + 2, kn.I32)]}
    change = {n: chains[v] if isinstance(v, str) else v for n, v in change.items()}
    with pytest.raises(kn.KernelError) as e:
        dense(kn, **change)
    assert e.value.status == kn.ERR_ARG and text in str(e.value)


def test_dense_lut_null_arguments(kn, rt):
    lib = rt.lib()
    assert lib.cvmk_dense_lut_prepare(None, None) == kn.ERR_ARG
    assert lib.cvmk_dense_lut_launch(None, None) == kn.ERR_ARG
    assert lib.cvmk_dense_lut_supported(None) == 0
    d, plan = kn.DenseLutDesc(rows=1, units=1, K=16, y_dtype=1, table_dtype=1, table_len=1), ct.create_string_buffer(ct.sizeof(kn.DenseLutPlan) + 64)
    assert lib.cvmk_dense_lut_supported(ct.byref(d)) == 1
    at = (ct.addressof(plan) + 63) // 64 * 64
    assert lib.cvmk_dense_lut_prepare(ct.byref(d), ct.c_void_p(at - 32 if at - 32 >= ct.addressof(plan) else at + 32)) == kn.ERR_ARG


def test_no_rows(kn):
    dense(kn, rows=0).launch()
    dense(kn, rows=0, x=0, y=0).launch()
    sample(kn, rows=0).launch()


def sample(kn, **change):
    a = dict(logits=1 << 20, rows=2, vocab=100, table=2 << 20, table_len=16, scale=3 << 20, random=4 << 20, token=5 << 20)
    a.update(change)
    return kn.Sample(**a)


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "sizes"), (dict(vocab=0), "sizes"), (dict(vocab=320 * 1024 + 1), "sizes"), (dict(table_len=0), "sizes"),
    (dict(pitch=99), "bad pitch"), (dict(pitch=-5), "bad pitch"), (dict(pitch=1 << 41), "bad pitch"),
    (dict(logits=0), "null operand"), (dict(table=0), "null operand"), (dict(scale=0), "null operand"), (dict(random=0), "null operand"),
    (dict(token=0), "null operand"),
] + [({n: (1 << 20) + 2}, "aligned") for n in ("logits", "table", "scale", "top_k", "top_p", "min_p", "random", "token", "weight", "kept")] +
    [(dict(mass=(1 << 20) + 4), "aligned")])
def test_sample_refuses(kn, change, text):
    with pytest.raises(kn.KernelError) as e:
        sample(kn, **change).launch()
    assert e.value.status == kn.ERR_ARG and text in str(e.value)


def test_sample_null_argument(kn, rt):
    assert rt.lib().cvmk_sample(None, None) == kn.ERR_ARG


def test_binding_matches_the_header(kn):
    """The sizes of the C structures: a plan begins with five 128-byte maps and is a whole number of 64 bytes."""
    assert ct.sizeof(kn.Chain) == 8 + 8 * 24
    assert ct.sizeof(kn.DenseLutDesc) == 4 * 8 + 3 * 8 + 4 * 4 + 8 + 2 * 4 + 8 + 2 * 4 + 3 * ct.sizeof(kn.Chain)
    assert kn.DenseLutPlan.kernel.offset == 640 + ct.sizeof(kn.DenseLutDesc)
    assert ct.sizeof(kn.SampleDesc) == 8 + 8 + 4 * 2 + 8 + 4 * 2 + 9 * 8
