"""The 4-bit-weight entry points without a GPU: argument checks of the C ABI (before any CUDA call),
packed sizes, workspace sizes, and the binding's refusals."""
import ctypes

import pytest
import torch

from gpu_pipes_b200 import _lib as L
from gpu_pipes_b200 import cuda_ext

P = ctypes.c_void_p
BASE = 1 << 32


def spec(k=1024, n=4096, group=128, dtype=L.GP_BF16, zeros=0):
    return L.GpW4Spec(k, n, group, dtype, zeros)


def nbytes(*a, **kw):
    return L.lib().gp_w4_packed_bytes(ctypes.byref(spec(*a, **kw)))


@pytest.mark.parametrize("k,n,group,zeros", [(8, 1, 32, 0), (64, 16, 64, 1), (1000, 17, 128, 0),
                                             (1024, 4096, 128, 0), (5128, 11003, 32, 1), (65536, 3, 64, 1)])
def test_packed_bytes(k, n, group, zeros):
    cells = -(-n // 16) * -(-k // 128)  # 16 columns x 128 rows
    want = cells * (1024 + 16 * (128 // group) * (4 if zeros else 2))
    assert nbytes(k, n, group, L.GP_F16, zeros) == want


def test_spec_refusals():
    lib = L.lib()
    assert lib.gp_w4_packed_bytes(None) == L.GP_ERR_ARG
    assert nbytes(k=0) == L.GP_ERR_SHAPE
    assert nbytes(k=-8) == L.GP_ERR_SHAPE
    assert nbytes(k=1001) == L.GP_ERR_SHAPE
    assert nbytes(k=65544) == L.GP_ERR_SHAPE
    assert nbytes(n=0) == L.GP_ERR_SHAPE
    assert nbytes(n=2**24 + 1) == L.GP_ERR_SHAPE
    assert nbytes(group=16) == L.GP_ERR_UNSUPPORTED
    assert nbytes(group=1024) == L.GP_ERR_UNSUPPORTED
    assert nbytes(dtype=2) == L.GP_ERR_ARG
    assert nbytes(k=65536, n=2**24) > 2**39  # sizes are 64-bit


def test_weight_entry_points_refuse():
    lib = L.lib()
    s = ctypes.byref(spec(128, 64))
    size = nbytes(128, 64)
    w, p = BASE, 2 * BASE
    assert lib.gp_w4_quantize_out(s, None, P(p), None) == L.GP_ERR_ARG
    assert lib.gp_w4_quantize_out(s, P(w), None, None) == L.GP_ERR_ARG
    assert lib.gp_w4_quantize_out(s, P(w), P(p + 8), None) == L.GP_ERR_ALIGN
    assert lib.gp_w4_quantize_out(s, P(w + 1), P(p), None) == L.GP_ERR_ALIGN
    assert lib.gp_w4_quantize_out(s, P(w), P(w + 128 * 64 * 2 - 16), None) == L.GP_ERR_ARG  # overlap
    assert "overlaps" in L.last_error()
    assert lib.gp_w4_dequantize_out(s, P(p), None, None) == L.GP_ERR_ARG
    assert lib.gp_w4_dequantize_out(s, P(p), P(p + size - 2), None) == L.GP_ERR_ARG
    assert lib.gp_w4_pack_out(s, None, P(w), None, P(p), None) == L.GP_ERR_ARG
    assert lib.gp_w4_pack_out(s, P(w), None, None, P(p), None) == L.GP_ERR_ARG
    assert lib.gp_w4_pack_out(s, P(w), P(3 * BASE), P(4 * BASE), P(p), None) == L.GP_ERR_ARG  # no zero points
    z = ctypes.byref(spec(128, 64, zeros=1))
    assert lib.gp_w4_pack_out(z, P(w), P(3 * BASE), None, P(p), None) == L.GP_ERR_ARG
    assert lib.gp_w4_pack_out(z, P(w), P(3 * BASE + 1), P(4 * BASE), P(p), None) == L.GP_ERR_ALIGN
    assert lib.gp_w4_unpack_out(s, P(p), None, None, None, None) == L.GP_ERR_ARG
    assert lib.gp_w4_unpack_out(s, P(p), None, None, P(w), None) == L.GP_ERR_ARG
    assert lib.gp_w4_unpack_out(z, P(p), P(w), P(w + 64), None, None) == L.GP_ERR_ARG  # codes and scales overlap


def _linear(m=4, act=0, x=BASE, packed=2 * BASE, bias=None, out=3 * BASE, s=None):
    s = s if s is not None else spec(128, 64)
    return L.lib().gp_w4_linear_out(ctypes.byref(s), m, act, P(x), P(packed), None if bias is None else P(bias),
                                    P(out), None)


def test_linear_refusals():
    assert _linear(m=0) == L.GP_OK  # nothing to do, no device touched
    assert _linear(m=-1) == L.GP_ERR_ARG
    assert _linear(m=2**31) == L.GP_ERR_SHAPE
    assert _linear(act=5) == L.GP_ERR_ARG
    assert _linear(x=0) == L.GP_ERR_ARG
    assert _linear(out=0) == L.GP_ERR_ARG
    assert _linear(packed=0) == L.GP_ERR_ARG
    assert _linear(x=BASE + 8) == L.GP_ERR_ALIGN
    assert _linear(out=3 * BASE + 1) == L.GP_ERR_ALIGN
    assert _linear(bias=4 * BASE + 1) == L.GP_ERR_ALIGN
    assert _linear(out=BASE) == L.GP_ERR_ARG
    assert _linear(out=2 * BASE + 16) == L.GP_ERR_ARG
    assert _linear(bias=3 * BASE + 2) == L.GP_ERR_ARG


def _mlp(widths=(1024, 4096, 1024), acts=(2, 0), tail=L.TAIL_RESIDUAL_LN, m=3, group=128, x=BASE, out=2 * BASE,
         packed=None, b=None, gamma=None, ws=5 * BASE, ws_bytes=None, skip=0, s=None):
    s = s if s is not None else L.make_spec(widths, acts, tail, L.GP_BF16, 1e-5, skip)
    n = s.n_layers
    packed = packed if packed is not None else [(16 + i) * BASE for i in range(n)]
    pp = (P * n)(*packed)
    bp = None if b is None else (P * n)(*b)
    if ws_bytes is None:
        ws_bytes = max(0, L.lib().gp_w4_mlp_workspace_bytes(ctypes.byref(s), m))
    return L.lib().gp_w4_mlp_out(ctypes.byref(s), group, 0, m, P(x), pp, bp, None if gamma is None else P(gamma),
                                 None, P(out), P(ws), ws_bytes, None)


def _ws(widths, tail, m, acts=None):
    s = L.make_spec(widths, acts or [0] * (len(widths) - 1), tail, L.GP_F16)
    return L.lib().gp_w4_mlp_workspace_bytes(ctypes.byref(s), m)


def test_mlp_workspace_bytes():
    assert _ws([64, 32], L.TAIL_NONE, 5) == 0
    assert _ws([64, 40], L.TAIL_LAYERNORM, 5) == 1024  # 5 x 40 fp32 = 800, in 256-byte pieces
    assert _ws([64, 200, 64], L.TAIL_NONE, 5) == 2048  # one hidden buffer: 2,000
    assert _ws([64, 200, 80, 40, 64], L.TAIL_NONE, 5) == 2 * 4096  # two that alternate, of two T per value
    assert _ws([1024, 4096, 1024], L.TAIL_RESIDUAL_LN, 2**20) == 2**20 * (4096 * 2 + 1024 * 4)
    assert _ws([8, 8, 8], L.TAIL_NONE, 2**30) == 2**30 * 16
    assert _ws([8, 8, 8, 8], L.TAIL_NONE, 2**30) == L.GP_ERR_SHAPE  # rows of two T are counted in 31 bits
    assert _ws([64, 200, 64], L.TAIL_NONE, -1) == L.GP_ERR_ARG
    assert _ws([64, 201, 64], L.TAIL_NONE, 1) == L.GP_ERR_SHAPE
    assert _ws([64, 200, 7], L.TAIL_NONE, 1) == 512  # the last width is free without a tail
    assert _ws([64, 200, 7], L.TAIL_LAYERNORM, 1) == L.GP_ERR_SHAPE
    assert _ws([64, 200, 72], L.TAIL_RESIDUAL_LN, 1) == L.GP_ERR_SHAPE


def test_mlp_refusals():
    assert _mlp(m=0) == L.GP_OK
    assert _mlp(m=-1) == L.GP_ERR_ARG
    assert _mlp(skip=1) == L.GP_ERR_UNSUPPORTED
    assert _mlp(acts=(7, 0)) == L.GP_ERR_ARG
    assert _mlp(group=48) == L.GP_ERR_UNSUPPORTED
    assert _mlp(x=0) == L.GP_ERR_ARG
    assert _mlp(packed=[16 * BASE, 0]) == L.GP_ERR_ARG
    assert _mlp(packed=[16 * BASE, 17 * BASE + 8]) == L.GP_ERR_ALIGN
    assert _mlp(x=BASE + 4) == L.GP_ERR_ALIGN
    assert _mlp(out=2 * BASE + 2) == L.GP_ERR_ALIGN
    assert _mlp(gamma=6 * BASE + 4) == L.GP_ERR_ALIGN
    assert _mlp(ws_bytes=100) == L.GP_ERR_ARG
    assert "workspace" in L.last_error()
    assert _mlp(ws=0) == L.GP_ERR_ARG
    assert _mlp(ws=5 * BASE + 8) == L.GP_ERR_ALIGN
    assert _mlp(ws=BASE) == L.GP_ERR_ARG  # workspace over x
    assert _mlp(ws=2 * BASE) == L.GP_ERR_ARG  # over out
    assert _mlp(out=16 * BASE) == L.GP_ERR_ARG  # out over weights
    assert _mlp(out=BASE + 2048) == L.GP_ERR_ARG  # shifted over x
    assert _mlp(tail=L.TAIL_NONE, out=BASE) == L.GP_ERR_ARG  # in place only with a tail
    s = L.make_spec((64, 64), (0,), 3, L.GP_F16)
    assert _mlp(s=s) == L.GP_ERR_ARG  # unknown tail


def test_binding_refusals():
    codes = torch.zeros(64, 32, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA"):
        cuda_ext.w4_pack(codes, torch.zeros(1, 32, dtype=torch.float16), group=64)
    with pytest.raises(RuntimeError, match="CUDA"):
        cuda_ext.w4_quantize(torch.zeros(64, 32, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        cuda_ext.W4Weight.empty(64, 32, 64, torch.float32, False, "cpu")
    with pytest.raises(L.GpError):
        cuda_ext.W4Weight.empty(63, 32, 64, torch.float16, False, "cpu")
    with pytest.raises(L.GpError):
        cuda_ext.W4Weight.empty(64, 32, 48, torch.float16, False, "cpu")
    w = cuda_ext.W4Weight.empty(64, 32, 64, torch.float16, False, "cpu")
    assert w.shape == (64, 32) and w.packed.numel() == nbytes(64, 32, 64, L.GP_F16, 0)
    with pytest.raises(RuntimeError, match="CUDA"):
        cuda_ext.w4_linear(torch.zeros(1, 64, dtype=torch.float16), w)
    with pytest.raises(RuntimeError, match="W4Weight"):
        cuda_ext.w4_linear_out(torch.zeros(1, 64), torch.zeros(64, 32), None, torch.zeros(1, 32))
    with pytest.raises(RuntimeError, match="none"):  # a chain mixes packed and plain weights
        cuda_ext.fused_mlp_out(torch.zeros(1, 64), [w, torch.zeros(32, 64)], [None, None], torch.zeros(1, 64),
                               acts=[0, 0])
    with pytest.raises(RuntimeError, match="skip_layer"):
        cuda_ext.fused_mlp_out(torch.zeros(1, 64), [w, w], [None, None], torch.zeros(1, 64), acts=[0, 0],
                               skip_layer=1)
    with pytest.raises(RuntimeError, match="match"):
        cuda_ext.w4_mlp_out(torch.zeros(1, 64), [w], [None], torch.zeros(1, 32), acts=[0, 0])


def test_chain_descriptions_hold_the_value_of_an_epsilon():
    """A tensor as the epsilon counts with its value at the call, in 16-bit and in 4-bit chains."""
    eps = torch.tensor(1.0)
    for value in (1.0, 0.5, 8.0):
        eps.fill_(value)
        assert cuda_ext._spec((64, 64), (0,), L.TAIL_LAYERNORM, L.GP_F16, eps, 0).ln_eps == value
        assert cuda_ext._w4_chain(2, (64, 64), (0,), L.TAIL_LAYERNORM, torch.float16, eps)[0]._obj.ln_eps == value
