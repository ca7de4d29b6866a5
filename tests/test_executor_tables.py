"""The tables of table-activated dense layers as the executor lays them out at load, on a device made of host memory
(tests/executor_host) whose small copies from pageable memory land after the call, as the CUDA runtime's may."""
import os
import shutil
import subprocess

import numpy as np
import pytest

from test_executor_host import CUDA, HOST, ROOT, SRC, put


@pytest.fixture(scope="module")
def load(tmp_path_factory):
    if shutil.which("g++") is None or not os.path.exists(os.path.join(CUDA, "cuda_runtime.h")):
        pytest.skip("no host compiler or CUDA headers")
    out = tmp_path_factory.mktemp("lut")
    srcs = [os.path.join(HOST, f) for f in ("ops.cc", "graph.cc", "host_pool.cc", "executor.cc", "c_api.cc")] + [os.path.join(SRC, f) for f in ("fake_device.cc", "lut.cc")]
    inc = os.path.join(ROOT, "include")
    flags = ["-std=c++17", "-O0", "-g1", "-fsanitize=address", "-pthread", "-I" + CUDA, "-I" + inc, "-I" + HOST]
    objs = [str(out / (os.path.basename(s) + ".o")) for s in srcs]
    procs = [subprocess.Popen(["g++"] + flags + ["-c", s, "-o", o]) for s, o in zip(srcs, objs)]
    assert all([p.wait() == 0 for p in procs])
    subprocess.check_call(["g++", "-fsanitize=address", "-pthread", "-Wl,--wrap=cudaMemcpy"] + objs + ["-o", str(out / "lut")])

    def run(work, when):
        p = subprocess.run([str(out / "lut"), when], cwd=work, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=60,
                           env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0:alloc_dealloc_mismatch=0"))
        assert p.returncode == 0, p.stderr[-4000:]
        return [np.array(line.split("=")[1].split(","), np.int64) for line in p.stdout.split() if line.startswith("@")]
    return run


def model(wl, table, precision, shifted):
    """A gated block with the table; `shifted`: a shift between the table and the product, through which the entries go at load."""
    g = wl.GraphBuilder(3)
    x = g.var("data", (4, 64), 8)
    shape = (4, 48)
    gate = g.lut(g.dense(x, 48, 9), table, precision, len(table) // 2)
    if shifted:
        gate = g.op("cvm_right_shift", [gate], shape, {"precision": 8, "shift_bit": 9})
    y = g.op("broadcast_mul", [gate, g.dense(x, 48, 9)], shape)
    js, pb = g.finish(g.op("cvm_right_shift", [y], shape, {"precision": 8, "shift_bit": 7}))
    return js, pb, np.zeros((4, 64), np.int8)


# (the fake device's element-wise kernel copies, to 8 bits behind a shift to 8: what it leaves is the table as it was when it ran)
@pytest.mark.parametrize("when", ["late", "early"])
@pytest.mark.parametrize("shifted", [False, True])
@pytest.mark.parametrize("table,precision", [(np.arange(256) * 300 - 30000, 17), (np.arange(200) - 100, 8), (np.arange(30000) - 9000, 17)])
def test_the_table_of_a_launch(load, wl, tmp_path, when, shifted, table, precision):
    table = table.astype(np.int8 if precision <= 8 else np.int32)
    put(tmp_path, *model(wl, table, precision, shifted))
    (got,) = load(tmp_path, when)
    assert np.array_equal(got, table.astype(np.int8) if shifted else table)
