"""The feed-forward products without a GPU: what the C entry points and the Python operators refuse, buffer sizes, and the modules' plain path."""
import ctypes

import pytest
import torch

from proteusai_b200 import _lib, build
from proteusai_b200.utils.model_utils.base_modules import fused_ops
from proteusai_b200.utils.model_utils.base_modules.base_modules import MLP, GatedMLP
from proteusai_b200.utils.model_utils.base_modules.encoder import Encoder, ProteusEncoderModel

OK, NULL, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE = 0, -1, -2, -3, -4, -5
P, ODD, HALFWAY = 0x10000, 0x10001, 0x10008  # addresses that are never used: aligned, at an odd byte, at 8 bytes


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def _linear_fwd(lib, **kw):
    a = dict(x=P, ldx=64, w=P, ldw=64, bias=P, fp32=0, r=P, ldr=32, y=P, ldy=32, saved=None, m=8, n=32, k=64, act=1, dtype=0)
    a.update(kw)
    return lib.pai_linear_fwd(a["x"], a["ldx"], a["w"], a["ldw"], a["bias"], a["fp32"], a["r"], a["ldr"], a["y"], a["ldy"], a["saved"], a["m"], a["n"],
                              a["k"], a["act"], a["dtype"], None)


def test_linear_forward_refusals(lib):
    f = lambda **kw: _linear_fwd(lib, **kw)
    for name in ("x", "w", "y"):
        assert f(**{name: None}) == NULL
    for name, value in (("m", -1), ("m", 1 << 31), ("n", 0), ("k", 0), ("n", (1 << 20) + 1), ("k", (1 << 20) + 1), ("ldx", 56), ("ldw", 56),
                        ("ldy", 31), ("ldr", -1)):
        assert f(**{name: value}) == SHAPE, (name, value)
    for name, value in (("x", HALFWAY), ("w", HALFWAY), ("ldx", 68), ("ldw", 68), ("y", ODD), ("r", ODD), ("bias", ODD), ("saved", HALFWAY)):
        assert f(**{name: value}) == ALIGN, (name, value)
    assert f(bias=P + 2, fp32=1) == ALIGN
    for name, value in (("act", -1), ("act", 5), ("dtype", 2), ("dtype", -1)):
        assert f(**{name: value}) == UNSUPPORTED, (name, value)


def _gated_bwd(lib, **kw):
    a = dict(dy=P, ldy=32, x=P, ldx=64, w=P, ldw=64, u=P, ldu=64, saved=P, dx=P, lddx=64, dw=P, du=P, db=P, dbu=P, fp32=0, ws=P, size=1 << 40, m=8,
             n=32, k=64, act=2, dtype=0)
    a.update(kw)
    return lib.pai_gated_bwd(*[a[i] for i in ("dy", "ldy", "x", "ldx", "w", "ldw", "u", "ldu", "saved", "dx", "lddx", "dw", "du", "db", "dbu", "fp32",
                                              "ws", "size", "m", "n", "k", "act", "dtype")], None)


def _linear_bwd(lib, **kw):
    a = dict(dy=P, ldy=32, x=P, ldx=64, w=P, ldw=64, saved=P, dx=P, lddx=64, dw=P, db=P, fp32=0, ws=P, size=1 << 40, m=8, n=32, k=64, act=1, dtype=0)
    a.update(kw)
    return lib.pai_linear_bwd(*[a[i] for i in ("dy", "ldy", "x", "ldx", "w", "ldw", "saved", "dx", "lddx", "dw", "db", "fp32", "ws", "size", "m", "n",
                                               "k", "act", "dtype")], None)


@pytest.mark.parametrize("call", (_linear_bwd, _gated_bwd))
def test_backward_refusals(lib, call):
    f = lambda **kw: call(lib, **kw)
    for name in ("dy", "x", "w", "saved", "ws"):
        assert f(**{name: None}) == NULL, name
    for name, value in (("m", 0), ("m", -1), ("n", 0), ("k", 0), ("ldx", 56), ("ldw", 56), ("lddx", 63), ("ldy", -1)):
        assert f(**{name: value}) == SHAPE, (name, value)
    for name, value in (("x", HALFWAY), ("w", HALFWAY), ("ldx", 68), ("saved", HALFWAY), ("ws", P + 128), ("dw", ODD), ("db", ODD), ("dx", ODD)):
        assert f(**{name: value}) == ALIGN, (name, value)
    gated = call is _gated_bwd
    need = lib.pai_dense_bwd_workspace_bytes(8, 32, 64, gated)
    assert need > 0 and f(size=need - 1) == WORKSPACE
    assert f(act=7) == UNSUPPORTED and f(dtype=2) == UNSUPPORTED


def test_gradient_without_activation_is_an_operand(lib):
    f = lambda **kw: _linear_bwd(lib, act=0, saved=None, **kw)
    assert f(dy=HALFWAY) == ALIGN and f(ldy=36) == ALIGN and f(ldy=24) == SHAPE
    assert _linear_bwd(lib, dy=HALFWAY, size=0) == WORKSPACE  # with an activation it may have any alignment: the next check speaks


def test_gated_forward_and_copy_refusals(lib):
    g = lambda x=P, w=P, u=P, h=P, ldu=64, ldh=32, m=8, act=2: lib.pai_gated_fwd(x, 64, w, 64, u, ldu, None, None, 0, h, ldh, None, m, 32, 64, act, 0,
                                                                                None)
    assert g(x=None) == g(w=None) == g(u=None) == g(h=None) == NULL
    assert g(ldu=56) == g(ldh=31) == g(m=-1) == SHAPE
    assert g(u=HALFWAY) == g(ldu=68) == g(h=ODD) == ALIGN
    assert g(act=9) == UNSUPPORTED
    arr = lambda t, *v: (t * len(v))(*v)

    def c(count=1, src=P, ld=7, dst=P, ldd=8, rows=4, cols=7):
        return lib.pai_copy_rows16(count, arr(ctypes.c_void_p, src), arr(ctypes.c_int64, ld), arr(ctypes.c_void_p, dst), arr(ctypes.c_int64, ldd),
                                   arr(ctypes.c_longlong, rows), arr(ctypes.c_int, cols), None)
    assert c(count=0) == c(count=4) == c(rows=-1) == c(cols=0) == c(ldd=0) == SHAPE
    assert c(src=None) == c(dst=None) == NULL
    assert c(src=ODD) == c(dst=HALFWAY) == c(ldd=12) == ALIGN


def test_buffer_sizes(lib):
    blocks = lambda m, n: ((m + 31) // 32) * ((n + 31) // 32)
    assert lib.pai_dense_saved_bytes(1, 1, 1, 0, 0) == 4096                      # a few tokens: fp32, whole blocks of 32 x 32
    assert lib.pai_dense_saved_bytes(5, 70, 64, 1, 0) == 2 * blocks(5, 70) * 4096
    big = blocks(65536, 2048)
    assert lib.pai_dense_saved_bytes(65536, 2048, 512, 0, 0) == big * (2048 + 64)   # bf16: fp16 and an exponent per 16 columns
    assert lib.pai_dense_saved_bytes(65536, 2048, 512, 1, 1) == 2 * big * 4096      # fp16: fp32
    assert lib.pai_dense_saved_bytes(0, 32, 64, 0, 0) == 0 and lib.pai_dense_saved_bytes(8, 32, 0, 0, 0) == 0
    assert lib.pai_dense_saved_bytes(8, 32, 64, 0, 3) == 0 and lib.pai_dense_bwd_workspace_bytes(8, 0, 64, 0) == 0
    # the gradient of the pre-activations (rows padded to 8 columns) is the least of the workspace
    assert lib.pai_dense_bwd_workspace_bytes(1000, 2001, 512, 1) >= 2 * 1000 * 2008 * 2


def test_python_refuses_cpu_tensors_and_unknown_activations():
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_ops.linear(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_ops.gated_linear(x, w, w)
    for f in (lambda act: fused_ops.linear(x, w, act=act), lambda act: fused_ops.gated_linear(x, w, w, act=act)):
        with pytest.raises(ValueError, match="act must be"):
            f("tanh")
    assert not fused_ops.dense_usable(x, w)


def test_modules_without_a_gpu_are_the_plain_blocks():
    torch.manual_seed(0)
    x = torch.randn(2, 5, 16)
    plain, fused = MLP(16, 16, 32, 1, 0.0), MLP(16, 16, 32, 1, 0.0, fused=True)
    assert set(plain.state_dict()) == set(fused.state_dict())
    fused.load_state_dict(plain.state_dict())
    assert torch.equal(plain(x), fused(x)) and torch.equal(plain(x) + x, fused(x, x))
    g = GatedMLP(16, 12, 32, dropout=0.0, act="gelu")
    h = torch.nn.functional.gelu(x @ g.gate_proj.weight.T + g.gate_proj.bias) * (x @ g.up_proj.weight.T + g.up_proj.bias)
    assert torch.allclose(g(x), h @ g.out_proj.weight.T + g.out_proj.bias, atol=1e-6)
    assert set(GatedMLP(16, 12, 32, bias=False).state_dict()) == {"gate_proj.weight", "up_proj.weight", "out_proj.weight"}
    with pytest.raises(ValueError):
        GatedMLP(act="tanh")


def test_encoder_options():
    assert isinstance(Encoder(64, 1, d_hidden=96).ffn, MLP) and not Encoder(64, 1, d_hidden=96).ffn.fused
    assert Encoder(64, 1, d_hidden=96, ffn="fused").ffn.fused
    assert set(Encoder(64, 1, d_hidden=96).state_dict()) == set(Encoder(64, 1, d_hidden=96, ffn="fused").state_dict())
    assert isinstance(Encoder(64, 1, d_hidden=96, ffn="gated").ffn, GatedMLP)
    assert isinstance(ProteusEncoderModel(64, 1, 1, 96, ffn="gated").encoders[0].ffn, GatedMLP)
    with pytest.raises(ValueError):
        Encoder(64, 1, ffn="none")
    with pytest.raises(ValueError):
        Encoder(64, 1, ffn="gated", hidden_layers=1)
