"""The microscaled calls of perf/operators.py without a GPU: every kind of case,
drawn or listed, has arguments that the library takes."""
import importlib.util
import os
import random

import pytest

import iris_testlib as tl

P = 1 << 20   # a 16-byte aligned address that nothing reads


@pytest.fixture(scope="module")
def ops():
    spec = importlib.util.spec_from_file_location("perf_operators", os.path.join(tl.ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


class Buffer:
    """A tensor's address and shape."""

    def __init__(self, rows, cols):
        self.shape = (rows, cols)

    def data_ptr(self):
        return P


def state(ops, c):
    """What prepare() makes of a case, without memory."""
    def codes(fmt, rows, cols):
        return (Buffer(rows, -(-cols // 128) * 128 // (2 if fmt == ops.FP4 else 1)), Buffer(rows, -(-cols // 512) * 16))
    s = {"case": c}
    if c["kind"] == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        s["aq"], s["as"] = codes(c["afmt"], m, k)
        s["wq"], s["ws"] = codes(ops.FP4, n, k)
        s["bias"] = Buffer(1, n)
        if c["epi"] == "swiglu_mx":
            s["q"], s["s"] = codes(ops.FP8, m, n // 2)
        else:
            s["out"] = Buffer(m, n // 2 if c["epi"] == "swiglu" else n)
        return s
    s["x"], s["w"], s["y"] = Buffer(c["rows"], c["cols"]), Buffer(1, c["cols"]), Buffer(c["rows"], c["cols"])
    s["q"], s["s"] = codes(c["fmt"], c["rows"], c["cols"])
    if c["kind"] == "norm" and c["add"] != "none":
        s["d"], s["gate"], s["x_out"] = (Buffer(c["rows"], c["cols"]) for _ in range(3))
    return s


def cases(ops):
    """The listed ones, drawn ones, and every combination of the choices."""
    rng = random.Random(1)
    yield from ops.listed()
    for _ in range(500):
        yield ops.draw(rng)
    for fmt in (ops.FP8, ops.FP4):
        for bf16 in (False, True):
            yield ops._quant(fmt, bf16, 5, 77)
        for add in ("none", "f32", "bf16"):
            for gate in (False, True):
                yield ops._norm(fmt, 5, 300, add, gate)
        for epi in ops.EPI:
            yield ops._gemm(fmt, epi, 5, 128, 300)


def test_arguments(ops):
    """A gate only beside the rows that it multiplies, those only with rows to
    write, one output per product: what the library does not refuse."""
    for c in cases(ops):
        a = ops._calls(state(ops, c))
        if c["kind"] == "norm":
            assert bool(a.gate) == (c["add"] != "none" and c["gate"]), c
            assert bool(a.d) == bool(a.x_out) == (c["add"] != "none"), c
        elif c["kind"] == "gemm":
            assert bool(a.out) != bool(a.mx_out.q), c
