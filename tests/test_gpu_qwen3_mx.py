"""The text encoder with microscaled linears (qwen3_model_quantize) against the
oracle on the weights that its 4-bit codes stand for: what differs is the
rounding of the linears' inputs to 8 bits.

A value's rounding to e4m3 is uniform within half a step, 2^-4 of its power of
two: 2.6e-2 of it in the mean square over a binade. A product's terms are
rounded independently, so its result carries the same share. The attention's
contribution carries two such roundings in a row (input, attention rows), the
MLP's those of its input, twice as gate and up are multiplied, of the product
and what the attention's error changes in the input: at most 4 x 2.6e-2 = 0.104
of what a layer adds to the stream."""
import ctypes
import os

import numpy as np
import pytest
from safetensors.torch import load_file

import iris_testlib as tl
import mx_reference as mx

pytestmark = pytest.mark.gpu
SHARD = "model-00001-of-00001.safetensors"


def dequantized_copy(src, dst):
    """A model directory with the linears' weights replaced by what their 4-bit rows stand for."""
    t = load_file(os.path.join(src, SHARD))
    out = []
    for name, v in t.items():
        x = v.float().numpy()
        if name.endswith("proj.weight"):
            code, s = mx.quantize(x, mx.FP4)
            x = mx.values(code, s, mx.FP4, x.shape[1]).astype(np.float32)
        out.append((name, tl.to_bf16(x).reshape(x.shape)))   # codes times powers of two are bf16 values
    os.makedirs(dst, exist_ok=True)
    tl.write_safetensors(os.path.join(dst, SHARD), out)
    for f in ("config.json", "model.safetensors.index.json"):
        with open(os.path.join(src, f)) as a, open(os.path.join(dst, f), "w") as b:
            b.write(a.read())


@pytest.fixture(scope="module")
def lib():
    lib = mx.bind(tl.hip())
    lib.qwen3_model_quantize.argtypes = [ctypes.c_void_p]
    return lib


@pytest.fixture(scope="module")
def dirs(tmp_path_factory):
    """A model of two layers, of which Z-Image's extraction runs the first, and its dequantized copy."""
    d = tmp_path_factory.mktemp("qwen3_mx")
    tl.write_qwen3_dir(str(d / "a"), hidden=320, inter=704, layers=2, seed=11)
    dequantized_copy(str(d / "a"), str(d / "b"))
    return str(d / "a"), str(d / "b")


def forward(lib, m, ids, mask, mode):
    lib.qwen3_model_set_extraction_mode(m, mode)
    width = lib.qwen3_model_text_dim(m)
    p = lib.qwen3_forward(m, ids.ctypes.data_as(tl.IP), mask.ctypes.data_as(tl.IP), len(ids))
    assert p, lib.iris_hip_last_error()
    out = np.ctypeslib.as_array(ctypes.cast(p, tl.FP), shape=(len(ids) * width,)).copy()
    ctypes.CDLL(None).free(ctypes.c_void_p(p))
    return out.reshape(len(ids), width)


@pytest.mark.parametrize("S,real", [(1, 1), (17, 17), (37, 20), (130, 130), (512, 90)])
def test_one_layer(lib, dirs, S, real):
    orc = tl.oracle()
    g, o = ctypes.c_void_p(lib.qwen3_model_load(dirs[0].encode())), ctypes.c_void_p(orc.orc_qwen3_load(dirs[1].encode()))
    assert lib.qwen3_model_quantize(g) == 0 and lib.qwen3_model_quantize(g) == 0
    rng = np.random.default_rng(S)
    ids, mask = rng.integers(0, 300, S).astype(np.int32), (np.arange(S) < real).astype(np.int32)
    got = forward(lib, g, ids, mask, 1)
    orc.orc_qwen3_set_mode(o, 1)
    want = tl.take_f32(orc, orc.orc_qwen3_forward(o, ids.ctypes.data_as(tl.IP), mask.ctypes.data_as(tl.IP), S, 0),
                       got.size).reshape(got.shape)
    emb = load_file(os.path.join(dirs[0], SHARD))["model.embed_tokens.weight"].float().numpy()[ids]
    a, b = got[:real] - emb[:real], want[:real] - emb[:real]
    assert np.isfinite(got).all()
    assert tl.rel_l2(a, b) < 0.104
    assert np.array_equal(forward(lib, g, ids, mask, 1), got)
    lib.qwen3_model_free(g)
    orc.orc_qwen3_free(o)


def test_all_layers_and_refusal(lib):
    """Flux's three extracted layers of a deep model: finite, the same bits every time, another length in between."""
    assert lib.qwen3_model_quantize(None) < 0
    m = ctypes.c_void_p(lib.qwen3_model_create_synthetic(256, 512, 4, 2, 28, 300, 5))
    assert lib.qwen3_model_quantize(m) == 0
    rng = np.random.default_rng(0)
    ids = rng.integers(0, 300, 512).astype(np.int32)
    one = np.ones(512, np.int32)
    a = forward(lib, m, ids, one, 0)
    forward(lib, m, ids[:40], one[:40], 0)
    assert np.isfinite(a).all() and np.array_equal(forward(lib, m, ids, one, 0), a)
    lib.qwen3_model_free(m)
