"""The text encoder with microscaled linears over several layers: what a layer
hands to the next one.

Layers add f32 sums to the stream, whether a norm follows (the product's f32
rows, added by the norm) or not (added by the product): one rounding of the same
sum, the same bits.

Against the oracle on the weights that the 4-bit codes stand for: one layer is
off by at most e = 0.104 of what it adds (test_gpu_qwen3_mx.py). The second
layer's input is then off by e |c1| of the stream's |x0 + c1|, and so by at most
e relative; a layer answers a relative change t of its input by at most 4 t of
what it adds: values and their weights (by queries and keys, one change each) 3
t in the attention, gate and up 2 t in the MLP, with the attention's among their
input's. So the sum of both is off by at most e |c1| + 5 e |c2|."""
import ctypes
import os

import numpy as np
import pytest
from safetensors.torch import load_file

import iris_testlib as tl
import mx_reference as mx
from test_gpu_qwen3_mx import SHARD, dequantized_copy, forward

gpu = pytest.mark.gpu


def signed_norms(d, seed):
    """The model's norm vectors with signs of their own: a wrong one gives other rows altogether."""
    rng = np.random.default_rng(seed)
    out = []
    for name, v in load_file(os.path.join(d, SHARD)).items():
        x = v.float().numpy()
        if name.endswith("layernorm.weight"):
            x = x * rng.choice([-1.0, 1.0], x.shape).astype(np.float32)
        out.append((name, tl.to_bf16(x).reshape(x.shape)))
    tl.write_safetensors(os.path.join(d, SHARD), out)


def swapped_copy(src, dst, a, b):
    """The model with two of its tensors exchanged."""
    os.makedirs(dst)
    out = []
    t = {k: v.float().numpy() for k, v in load_file(os.path.join(src, SHARD)).items()}
    t[a], t[b] = t[b], t[a]
    for name, x in t.items():
        out.append((name, tl.to_bf16(x).reshape(x.shape)))
    tl.write_safetensors(os.path.join(dst, SHARD), out)
    for f in ("config.json", "model.safetensors.index.json"):
        with open(os.path.join(src, f)) as i, open(os.path.join(dst, f), "w") as o:
            o.write(i.read())


@pytest.fixture(scope="module")
def dirs(tmp_path_factory):
    """Three layers, of which Z-Image's extraction runs the first two, and the dequantized copy."""
    d = tmp_path_factory.mktemp("qwen3_mx_layers")
    tl.write_qwen3_dir(str(d / "a"), hidden=320, inter=704, layers=3, seed=12)
    signed_norms(str(d / "a"), 3)
    dequantized_copy(str(d / "a"), str(d / "b"))
    for i, (p, q) in enumerate(WRONG):
        swapped_copy(str(d / "b"), str(d / f"w{i}"), p, q)
    return str(d / "a"), str(d / "b"), [str(d / f"w{i}") for i in range(len(WRONG))]


L = "model.layers.%d."
WRONG = [(L % 0 + "input_layernorm.weight", L % 1 + "input_layernorm.weight"),
         (L % 1 + "input_layernorm.weight", L % 2 + "input_layernorm.weight"),
         (L % 1 + "input_layernorm.weight", L % 1 + "post_attention_layernorm.weight"),
         (L % 0 + "mlp.down_proj.weight", L % 1 + "mlp.down_proj.weight")]


def streams(orc, d, ids, mask):
    """What the oracle's first layer adds to the embedding, and its second."""
    o = ctypes.c_void_p(orc.orc_qwen3_load(d.encode()))
    orc.orc_qwen3_set_mode(o, 1)
    emb = load_file(os.path.join(d, SHARD))["model.embed_tokens.weight"].float().numpy()[ids]
    run = lambda last: tl.take_f32(orc, orc.orc_qwen3_forward(  # noqa: E731
        o, ids.ctypes.data_as(tl.IP), mask.ctypes.data_as(tl.IP), len(ids), last), emb.size).reshape(emb.shape)
    # a limit of layer 0 leaves the extraction empty: the first layer alone is the model's with two layers
    two = run(-1)
    orc.orc_qwen3_free(o)
    return emb, two


def first_layer(orc, d, tmp, ids, mask):
    """The same model cut to two layers, of which the extraction runs one."""
    os.makedirs(tmp, exist_ok=True)
    for f in (SHARD, "model.safetensors.index.json"):
        if not os.path.exists(os.path.join(tmp, f)):
            os.symlink(os.path.join(d, f), os.path.join(tmp, f))
    with open(os.path.join(d, "config.json")) as i, open(os.path.join(tmp, "config.json"), "w") as o:
        o.write(i.read().replace('"num_hidden_layers": 3', '"num_hidden_layers": 2'))
    return streams(orc, tmp, ids, mask)


def inputs(S, real):
    rng = np.random.default_rng(S)
    return rng.integers(0, 300, S).astype(np.int32), (np.arange(S) < real).astype(np.int32)


def bound(orc, dirs, tmp, ids, mask, real):
    """The oracle's stream after two layers and how far it may be off."""
    emb, two = streams(orc, dirs[1], ids, mask)
    _, one = first_layer(orc, dirs[1], tmp, ids, mask)
    c1, c2 = (one - emb)[:real].astype(np.float64), (two - one)[:real].astype(np.float64)
    return two[:real], 0.104 * (np.linalg.norm(c1) + 5 * np.linalg.norm(c2))


SIZES = [(17, 17), (37, 20), (130, 130)]


@pytest.mark.parametrize("S,real", SIZES)
def test_the_bound_tells(dirs, tmp_path, S, real):
    """Without a GPU: a wrong norm vector or product between the layers is past the bound."""
    orc = tl.oracle()
    ids, mask = inputs(S, real)
    want, tol = bound(orc, dirs, str(tmp_path / "one"), ids, mask, real)
    for d in dirs[2]:
        assert np.linalg.norm(streams(orc, d, ids, mask)[1][:real] - want) > tol, d


@gpu
@pytest.mark.parametrize("S,real", SIZES)
def test_two_layers(dirs, tmp_path, S, real):
    orc, lib = tl.oracle(), mx.bind(tl.hip())
    lib.qwen3_model_quantize.argtypes = [ctypes.c_void_p]
    ids, mask = inputs(S, real)
    want, tol = bound(orc, dirs, str(tmp_path / "one"), ids, mask, real)
    g = ctypes.c_void_p(lib.qwen3_model_load(dirs[0].encode()))
    assert lib.qwen3_model_quantize(g) == 0
    got = forward(lib, g, ids, mask, 1)[:real]
    assert np.linalg.norm(got.astype(np.float64) - want) < tol
    lib.qwen3_model_free(g)


@gpu
@pytest.mark.parametrize("S", [1, 37, 300, 512])
def test_layers_hand_on_what_they_give(S):
    """Flux's extracted layers 8 and 17, which layers follow, are the last layers
    of models cut behind them, bit for bit."""
    lib = mx.bind(tl.hip())
    lib.qwen3_model_quantize.argtypes = [ctypes.c_void_p]
    ids, mask = inputs(S, S)
    h = 256

    def encode(layers, mode):
        m = ctypes.c_void_p(lib.qwen3_model_create_synthetic(h, 512, 4, 2, layers, 300, 5))
        assert lib.qwen3_model_quantize(m) == 0
        out = forward(lib, m, ids, mask, mode)
        lib.qwen3_model_free(m)
        return out
    flux = encode(28, 0)
    for slot, layer in enumerate((8, 17, 26)):
        assert np.array_equal(flux[:, slot * h:(slot + 1) * h], encode(layer + 2, 1)), layer
