"""Argument checks of the block norms, without a GPU."""
import ctypes

import pytest
import torch

from gpu_pipes_b200 import _lib as L
from gpu_pipes_b200 import cuda_ext

P = ctypes.c_void_p
B = 1 << 32


def call(m=4, width=64, dtype=L.GP_F16, x32=0, y32=0, post=0, pre=1, gate_rows=0, x=B, y=2 * B, gate=0, pg=0, pb=0,
         ng=0, nb=0, r=3 * B, h=4 * B):
    s = L.GpBlockNormSpec(width, dtype, x32, y32, post, pre, 1e-5, 1e-5, 1.0, 1.0, gate_rows)
    return L.lib().gp_block_norm_out(ctypes.byref(s), m, *[P(v) for v in (x, y, gate, pg, pb, ng, nb, r, h)], None)


def test_refusals():
    assert L.lib().gp_block_norm_out(None, 1, *[None] * 10) == L.GP_ERR_ARG
    assert call(m=0) == L.GP_OK
    assert call(m=0, x=0, y=2 * B) == L.GP_OK
    assert call(m=-1) == L.GP_ERR_ARG
    assert call(m=2**31) == L.GP_ERR_SHAPE
    for width in (0, -8, 12, 32776):
        assert call(width=width) == L.GP_ERR_SHAPE
    assert call(dtype=2) == L.GP_ERR_ARG
    assert call(post=3) == L.GP_ERR_ARG
    assert call(pre=-1) == L.GP_ERR_ARG
    assert call(gate_rows=-1) == L.GP_ERR_ARG
    assert call(x=0, y=0) == L.GP_ERR_ARG
    assert call(r=0, h=0) == L.GP_ERR_ARG
    assert call(y=0, post=2) == L.GP_ERR_ARG
    assert call(y=0, gate=5 * B) == L.GP_ERR_ARG
    for name in ("x", "y", "gate", "pg", "pb", "ng", "nb", "r", "h"):
        assert call(**{name: 9 * B + 8}) == L.GP_ERR_ALIGN, name


def test_overlaps():
    # 4 rows of 64: 512 bytes in 16 bits, 1,024 in 32
    assert call(h=3 * B) == L.GP_ERR_ARG  # r and h
    assert call(r=B + 128) == L.GP_ERR_ARG  # shifted over x
    assert call(h=2 * B + 496) == L.GP_ERR_ARG  # its last bytes over y's first
    assert call(x32=1, h=B) == L.GP_ERR_ARG  # 16-bit rows in place of 32-bit ones
    assert call(y32=1, r=2 * B) == L.GP_ERR_ARG
    assert call(gate=3 * B) == L.GP_ERR_ARG
    assert call(gate=3 * B - 128, gate_rows=2) == L.GP_ERR_ARG  # the second gate row is r
    assert call(ng=4 * B + 16) == L.GP_ERR_ARG
    assert "overlap" in L.last_error()


def test_binding_refusals():
    x = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        cuda_ext.block_norm(x, x, pre=L.NORM_RMS)
    with pytest.raises(RuntimeError, match="needs x or y"):
        cuda_ext.block_norm(None, None, pre=L.NORM_RMS)
    with pytest.raises(RuntimeError, match="r or h"):
        cuda_ext.block_norm(x, x, want_r=False)
    with pytest.raises(RuntimeError, match="dtype"):
        cuda_ext.block_norm(x.float(), x.float(), pre=L.NORM_RMS)
    with pytest.raises(RuntimeError, match="2-D"):
        cuda_ext.block_norm(x[0], pre=L.NORM_RMS)


def test_binding_refuses_32_bit_parameters_and_outputs():
    """With x and y in fp32 nothing else names the 16-bit type: a gate, a norm's parameters or an h in
    fp32 are refused by name, not read or written as 16-bit values."""
    x = torch.zeros(4, 64)
    row = torch.zeros(64)
    for name in ("gate", "post_gamma", "post_beta", "pre_gamma", "pre_beta"):
        with pytest.raises(RuntimeError, match=f"{name} must be float16 or bfloat16"):
            cuda_ext.block_norm(x, x, post=L.NORM_RMS, **{name: row})
    with pytest.raises(RuntimeError, match="h must be float16 or bfloat16"):
        cuda_ext.block_norm_out(x, x, None, torch.zeros(4, 64), pre=L.NORM_RMS)
    with pytest.raises(RuntimeError, match="h must be float16 or bfloat16"):
        cuda_ext.block_norm(x, x, pre=L.NORM_RMS, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="gate must be a tensor"):
        cuda_ext.block_norm(x, x, gate=[1.0] * 64)
    with pytest.raises(RuntimeError, match="CUDA"):  # nothing else amiss
        cuda_ext.block_norm(x, x)
