"""ctypes binding of the launchers of include/cvmk_kernels.h that a program calls beside a model: dense layers with a
table as their activation (cvmk_dense_lut_*) and sampling (cvmk_sample).

Operands are device addresses as plain integers (0: none), in the layouts the header describes; the caller keeps the
memory they point to.  A status other than CVMK_OK raises KernelError with the text of cvmk_last_error().
"""
import ctypes as ct

from . import runtime as _rt

OK, ERR_ARG, ERR_CUDA, ERR_UNSUPPORTED = 0, 1, 2, 3
I8, I32 = 1, 4
(RELU, RSHIFT, LSHIFT, CLIP, ADD_T, SUB_T, RSUB_T, ADD_C, MUL_S, ADD_S, RSUB_S, MAX_S, DIV_S, RDIV_S, GT_S, LT_S, ABS, NEG,
 PRECISION) = range(1, 20)
MAX_STEPS = 8
MAX_VOCAB = 320 * 1024


class KernelError(RuntimeError):
    """A launcher answered something else than CVMK_OK."""

    def __init__(self, status, what):
        super().__init__("%s returned status %d: %s" % (what, status, (_rt.lib().cvmk_last_error() or b"").decode("utf-8", "replace")))
        self.status = status


class _Step(ct.Structure):
    _fields_ = [("op", ct.c_int32), ("a", ct.c_int32), ("b", ct.c_int32), ("ptr_dtype", ct.c_int32), ("ptr", ct.c_void_p)]


class Chain(ct.Structure):
    """cvmk_epilogue, from steps as tuples: (op,), (op, a), (op, a, b), (ADD_C, address) or (ADD_T | SUB_T | RSUB_T, address, type)."""
    _fields_ = [("n", ct.c_int32), ("reserved", ct.c_int32), ("s", _Step * MAX_STEPS)]

    def __init__(self, steps=()):
        super().__init__()
        if len(steps) > MAX_STEPS:
            raise ValueError("a chain has at most %d steps" % MAX_STEPS)
        self.n = len(steps)
        for i, (op, *rest) in enumerate(steps):
            if op == ADD_C:
                self.s[i] = _Step(op, 0, 0, I32, rest[0])
            elif op in (ADD_T, SUB_T, RSUB_T):
                self.s[i] = _Step(op, 0, 0, rest[1], rest[0])
            else:
                self.s[i] = _Step(op, *(rest + [0, 0])[:2], 0, None)


class DenseLutDesc(ct.Structure):
    _fields_ = ([(n, ct.c_void_p) for n in ("x", "w", "v", "y")] + [(n, ct.c_int64) for n in ("x_pitch", "w_pitch", "y_pitch")] +
                [(n, ct.c_int32) for n in ("rows", "units", "K", "y_dtype")] + [("table", ct.c_void_p), ("table_len", ct.c_int32), ("table_dtype", ct.c_int32)] +
                [("status", ct.c_void_p), ("params_static", ct.c_int32), ("reserved", ct.c_int32)] + [(n, Chain) for n in ("chain_w", "chain_v", "chain_y")])


class DenseLutPlan(ct.Structure):
    _fields_ = ([(n, ct.c_uint8 * 128) for n in ("tmap_x", "tmap_w", "tmap_v", "tmap_y", "tmap_r")] + [("d", DenseLutDesc)] +
                [(n, ct.c_int32) for n in ("kernel", "grid", "smem_bytes", "stages", "split", "row_tile", "table_smem", "io", "device")] + [("reserved", ct.c_int32 * 3)])


class SampleDesc(ct.Structure):
    _fields_ = ([("logits", ct.c_void_p), ("pitch", ct.c_int64), ("rows", ct.c_int32), ("vocab", ct.c_int32), ("table", ct.c_void_p),
                 ("table_len", ct.c_int32), ("reserved", ct.c_int32)] +
                [(n, ct.c_void_p) for n in ("scale", "top_k", "top_p", "min_p", "random", "token", "weight", "mass", "kept")])


def _function(name, *args):
    f = _rt.lib()[name]   # (an object of its own, so that its declared types are nobody else's)
    f.argtypes, f.restype = list(args), ct.c_int
    return f


class DenseLut:
    """A prepared cvmk_dense_lut_* launch.  The plan is made for the device that is current now."""

    def __init__(self, x, w, table, y, rows, units, k, table_len, v=0, x_pitch=0, w_pitch=0, y_pitch=0, y_dtype=I8, table_dtype=I8,
                 chain_w=(), chain_v=(), chain_y=(), status=0, params_static=False):
        d = DenseLutDesc(x=x, w=w, v=v or None, y=y, x_pitch=x_pitch, w_pitch=w_pitch, y_pitch=y_pitch, rows=rows, units=units, K=k, y_dtype=y_dtype,
                         table=table, table_len=table_len, table_dtype=table_dtype, status=status or None, params_static=1 if params_static else 0)
        d.chain_w, d.chain_v, d.chain_y = Chain(chain_w), Chain(chain_v), Chain(chain_y)
        self._memory = ct.create_string_buffer(ct.sizeof(DenseLutPlan) + 64)
        self.plan = DenseLutPlan.from_buffer(self._memory, -ct.addressof(self._memory) % 64)
        status = _function("cvmk_dense_lut_prepare", ct.c_void_p, ct.c_void_p)(ct.addressof(d), ct.addressof(self.plan))
        if status != OK:
            raise KernelError(status, "cvmk_dense_lut_prepare")
        self._launch, self._at = _function("cvmk_dense_lut_launch", ct.c_void_p, ct.c_void_p), ct.addressof(self.plan)

    def launch(self, stream=0):
        """Enqueues the kernel on `stream`, a cudaStream_t as an integer."""
        status = self._launch(self._at, stream)
        if status != OK:
            raise KernelError(status, "cvmk_dense_lut_launch")


class Sample:
    """A cvmk_sample call with its arguments; launch() may be repeated as the operands' contents change."""

    def __init__(self, logits, rows, vocab, table, table_len, scale, random, token, pitch=0, top_k=0, top_p=0, min_p=0, weight=0, mass=0, kept=0):
        self.desc = SampleDesc(logits=logits, pitch=pitch, rows=rows, vocab=vocab, table=table, table_len=table_len, scale=scale, top_k=top_k or None,
                               top_p=top_p or None, min_p=min_p or None, random=random, token=token, weight=weight or None, mass=mass or None,
                               kept=kept or None)
        self._launch, self._at = _function("cvmk_sample", ct.c_void_p, ct.c_void_p), ct.addressof(self.desc)

    def launch(self, stream=0):
        """Enqueues the kernel on `stream`, a cudaStream_t as an integer."""
        status = self._launch(self._at, stream)
        if status != OK:
            raise KernelError(status, "cvmk_sample")
