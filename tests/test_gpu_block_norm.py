"""The block norms on the GPU against the definition in 64 bits.

Bounds: all arithmetic is fp32 on a row of H values. A sum of H values taken as at most 40 values per
thread, then 5 + 32 partial sums, is off by at most about 80 half steps of the sum of magnitudes; with
the few operations per element after it, C = 128 half steps bound each statistic and each element's
arithmetic, relative to the magnitudes that go into it. Stored values add one rounding."""
import os
import subprocess
import sys

import pytest
import torch

from gpu_pipes_b200 import _lib as L
from gpu_pipes_b200 import cuda_ext
from tests._tol import U32, check, rounded

pytestmark = pytest.mark.gpu
C = 128 * U32
NONE, LAYER, RMS = L.NORM_NONE, L.NORM_LAYER, L.NORM_RMS


def _norm(kind, v, err, gamma, beta, eps):
    """(N(v), bound of its error before a store) for v with an error bound err."""
    if kind == NONE:
        return v, err
    mean = v.mean(1, keepdim=True) if kind == LAYER else torch.zeros_like(v[:, :1])
    d = v - mean
    mag = v.abs() + mean.abs()
    e = err + err.mean(1, keepdim=True) + C * (mag + v.abs().mean(1, keepdim=True))
    rs = 1.0 / torch.sqrt(d.square().mean(1, keepdim=True) + eps)
    rel = 2 * torch.sqrt(e.square().mean(1, keepdim=True)) * rs + C
    g = gamma.double() if gamma is not None else torch.ones_like(v[0])
    b = beta.double() if beta is not None else torch.zeros_like(v[0])
    n = d * rs * g
    return n + b, e * rs * g.abs() + n.abs() * rel + C * (n.abs() + b.abs())


def _reference(x, y, post, pre, gate, pg, pb, ng, nb, xs, ys, pe, ne):
    xs, ys = torch.tensor(xs).double().item(), torch.tensor(ys).double().item()  # fp32 arguments
    base = x if x is not None else y
    r, err = torch.zeros_like(base, dtype=torch.float64), torch.zeros_like(base, dtype=torch.float64)
    if y is not None:
        v, e = _norm(post, y.double(), r.clone(), pg, pb, torch.tensor(pe).double().item())
        s = torch.full_like(v[:1], ys)
        if gate is not None:
            g = gate.double().reshape(-1, y.shape[1])
            s = s * g.repeat_interleave(y.shape[0] // g.shape[0], 0)
        r, err = v * s, e * s.abs() + C * (v * s).abs()
    if x is not None:
        r, err = r + xs * x.double(), err + C * (r.abs() + abs(xs) * x.double().abs())
    h, he = _norm(pre, r, err, ng, nb, torch.tensor(ne).double().item())
    return r, err, h, he


def _make(dev, m, h, dtype, stream, ydt, gates, seed=0):
    g = torch.Generator().manual_seed(1000 * m + h + seed)
    t = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (t(m, h) * 1.5 + 0.2).to(stream)
    y = (t(m, h) * 0.7 - 0.1).to(ydt)
    gate = None if gates == 0 else (t(h) if gates == 1 else t(gates, h)).to(dtype)
    params = [(t(h) * 0.1 + 1).to(dtype), (t(h) * 0.1).to(dtype), (t(h) * 0.1 + 1).to(dtype), (t(h) * 0.1).to(dtype)]
    return [v if v is None else v.to(dev) for v in (x, y, gate, *params)]


def _run_and_check(x, y, post, pre, gate, pg, pb, ng, nb, dtype, xs=1.0, ys=1.0, pe=1e-5, ne=1e-6):
    if post == NONE:
        pg = pb = None
    if pre == NONE:
        ng = nb = None
    r, h = cuda_ext.block_norm(x, y, post=post, pre=pre, gate=gate, post_gamma=pg, post_beta=pb, pre_gamma=ng,
                               pre_beta=nb, x_scale=xs, y_scale=ys, post_eps=pe, pre_eps=ne, dtype=dtype)
    rr, re, hh, he = _reference(x, y, post, pre, gate, pg, pb, ng, nb, xs, ys, pe, ne)
    if r is not None:
        check(r, rr, rounded(rr, re, r.dtype), "r")
    if h is not None:
        check(h, hh, rounded(hh, he, dtype), "h")
    return r, h


WIDTHS = [8, 16, 256, 264, 512, 1000, 1024, 1032, 2048, 2056, 4096, 4104, 8192, 8200, 16384, 16392, 32768]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_widths(cuda_dev, width, dtype):
    m = 11
    x, y, gate, pg, pb, ng, nb = _make(cuda_dev, m, width, dtype, dtype, dtype, 1)
    _run_and_check(x, y, RMS, LAYER, gate, pg, pb, ng, nb, dtype, xs=1.25, ys=0.7)


@pytest.mark.parametrize("post", [NONE, LAYER, RMS])
@pytest.mark.parametrize("pre", [NONE, LAYER, RMS])
@pytest.mark.parametrize("stream,ydt", [("16", "16"), ("32", "16"), ("16", "32"), ("32", "32")])
@pytest.mark.parametrize("width", [136, 2104])
def test_kinds_and_types(cuda_dev, post, pre, stream, ydt, width):
    for dtype in (torch.float16, torch.bfloat16):
        sd = torch.float32 if stream == "32" else dtype
        yd = torch.float32 if ydt == "32" else dtype
        x, y, gate, pg, pb, ng, nb = _make(cuda_dev, 12, width, dtype, sd, yd, 4)
        _run_and_check(x, y, post, pre, gate, pg, pb, ng, nb, dtype, xs=0.5, ys=2.0)


@pytest.mark.parametrize("m,gates", [(1, 0), (1, 1), (3, 3), (8, 2), (9, 1), (4099, 0), (70000, 7)])
@pytest.mark.parametrize("width", [64, 1088])
def test_rows_and_gates(cuda_dev, m, gates, width):
    dtype = torch.bfloat16
    x, y, gate, pg, pb, ng, nb = _make(cuda_dev, m, width, dtype, dtype, dtype, gates)
    _run_and_check(x, y, LAYER, RMS, gate, pg, None, ng, None, dtype)


def test_missing_operands(cuda_dev):
    dtype = torch.float16
    x, y, gate, pg, pb, ng, nb = _make(cuda_dev, 7, 520, dtype, dtype, dtype, 1)
    r, h = _run_and_check(x, None, NONE, LAYER, None, pg, pb, ng, nb, dtype)  # the first block's norm
    assert r is None
    _run_and_check(None, y, RMS, NONE, gate, pg, None, ng, nb, dtype)  # no residual
    _run_and_check(x, y, NONE, NONE, None, None, None, None, None, dtype)  # a plain residual add
    _run_and_check(x, y, RMS, RMS, None, None, None, None, None, dtype)  # no parameters
    # the C entry's h without a norm is r in 16 bits
    r = torch.empty(7, 520, dtype=torch.float32, device=cuda_dev)
    h = torch.empty(7, 520, dtype=dtype, device=cuda_dev)
    cuda_ext.block_norm_out(x.float(), y, r, h)
    assert torch.equal(h, r.to(dtype))
    empty = x[:0]
    r, h = cuda_ext.block_norm(empty, empty, pre=RMS)
    assert r.shape == h.shape == (0, 520)


def test_degenerate_rows(cuda_dev):
    """Rows of zeros, constants, a large offset, infinities and NaN: each follows the definition,
    and none changes another row."""
    dtype = torch.bfloat16
    x, y, gate, pg, pb, ng, nb = _make(cuda_dev, 9, 1048, dtype, dtype, dtype, 0)
    x[1], y[1] = 0, 0
    x[3], y[3] = 2.5, -1.0
    y[5] = y[5] * 0.01 + 300  # LayerNorm of a large offset: two-pass statistics
    clean = _run_and_check(x, y, LAYER, LAYER, None, pg, pb, ng, nb, dtype)
    xx, yy = x.clone(), y.clone()
    xx[0, 7] = float("nan")
    yy[2, 1047] = float("inf")
    yy[8, 0] = -float("inf")
    r, h = cuda_ext.block_norm(xx, yy, post=LAYER, pre=LAYER, post_gamma=pg, post_beta=pb, pre_gamma=ng,
                               pre_beta=nb, pre_eps=1e-6)
    keep = [1, 3, 4, 5, 6, 7]
    for got, want in zip((r, h), clean):
        assert torch.equal(got[keep], want[keep])
    assert h[0].isnan().all() and h[2].isnan().all() and h[8].isnan().all()
    assert r[0, 7].isnan() and not r[0, :7].isnan().any()


def test_in_place(cuda_dev):
    for width in (200, 1000, 4096):
        x, y, gate, pg, pb, ng, nb = _make(cuda_dev, 301, width, torch.float16, torch.float16, torch.float16, 1)
        kw = dict(post=RMS, pre=LAYER, gate=gate, post_gamma=pg, pre_gamma=ng, pre_beta=nb, x_scale=0.9)
        r, h = cuda_ext.block_norm(x, y, **kw)
        x2, y2 = x.clone(), y.clone()
        cuda_ext.block_norm_out(x2, y2, x2, y2, **kw)  # r over x, h over y
        assert torch.equal(x2, r) and torch.equal(y2, h)
        x3, y3 = x.clone(), y.clone()
        cuda_ext.block_norm_out(x3, y3, y3, x3, **kw)  # r over y, h over x
        assert torch.equal(y3, r) and torch.equal(x3, h)


def test_rows_behind_the_last_stay(cuda_dev):
    x, y, *_ = _make(cuda_dev, 5, 264, torch.float16, torch.float16, torch.float16, 0)
    r = torch.full((8, 264), 7.0, dtype=torch.float16, device=cuda_dev)
    h = r.clone()
    cuda_ext.block_norm_out(x, y, r[:5], h[:5], pre=RMS)
    assert (r[5:] == 7).all() and (h[5:] == 7).all()


def test_same_result_every_time_and_on_another_stream(cuda_dev):
    x, y, gate, pg, pb, ng, nb = _make(cuda_dev, 333, 5000, torch.bfloat16, torch.float32, torch.bfloat16, 1)
    kw = dict(post=RMS, pre=LAYER, gate=gate, post_gamma=pg, pre_gamma=ng)
    first = cuda_ext.block_norm(x, y, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cuda_ext.block_norm(x, y, **kw)
    side.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)


def test_binding_refusals_on_device(cuda_dev):
    x, y, gate, pg, pb, ng, nb = _make(cuda_dev, 6, 64, torch.float16, torch.float16, torch.float16, 4)
    with pytest.raises(RuntimeError, match="multiple of 4 gate rows"):
        cuda_ext.block_norm(x, y, pre=RMS, gate=gate)
    with pytest.raises(RuntimeError, match="contiguous"):
        cuda_ext.block_norm(x[:, ::2], y[:, ::2], pre=RMS)
    with pytest.raises(RuntimeError, match="must be torch.float16"):
        cuda_ext.block_norm(x, y.bfloat16(), pre=RMS, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="shape"):
        cuda_ext.block_norm(x, y[:5], pre=RMS)
    with pytest.raises(RuntimeError, match="post_gamma"):
        cuda_ext.block_norm(x, y, post=RMS, post_gamma=pg[:32])
    with pytest.raises(L.GpError, match="16-byte"):
        flat = torch.zeros(64 * 6 + 4, dtype=torch.float16, device=cuda_dev)
        cuda_ext.block_norm(flat[4:].view(6, 64), pre=RMS)
    with pytest.raises(L.GpError, match="multiple of 8"):
        cuda_ext.block_norm(torch.zeros(6, 60, dtype=torch.float16, device=cuda_dev), pre=RMS)


def test_first_call_of_a_process_may_be_captured(cuda_dev):
    # the norms and the conversions of weights allocate nothing, not even on their first call
    code = """if True:
        import torch
        import __graft_entry__ as e
        e.load_package()
        from gpu_pipes_b200 import _lib as L, cuda_ext
        x = torch.randn(5, 256, device="cuda").half()
        w = torch.randn(256, 64, device="cuda").half()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _, h = cuda_ext.block_norm(x, pre=L.NORM_RMS)
            d = cuda_ext.w4_dequantize(cuda_ext.w4_quantize(w))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, cuda_ext.block_norm(x, pre=L.NORM_RMS)[1])
        assert torch.equal(d, cuda_ext.w4_dequantize(cuda_ext.w4_quantize(w)))
        print("captured")
    """
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_all_in_32_bits(cuda_dev):
    """x, y and r in fp32 and nothing in 16 bits: the sums and norms that need no parameters run; fp32
    parameters, gates and normed rows are refused."""
    x, y, gate, pg, pb, ng, nb = _make(cuda_dev, 6, 264, torch.float16, torch.float32, torch.float32, 1)
    _run_and_check(x, y, LAYER, NONE, None, None, None, None, None, torch.float16, xs=0.5, ys=2.0)
    with pytest.raises(RuntimeError, match="gate must be float16 or bfloat16"):
        cuda_ext.block_norm(x, y, gate=gate.float())
    with pytest.raises(RuntimeError, match="post_gamma must be float16 or bfloat16"):
        cuda_ext.block_norm(x, y, post=RMS, post_gamma=pg.float())
    with pytest.raises(RuntimeError, match="h must be float16 or bfloat16"):
        cuda_ext.block_norm_out(x, y, torch.empty_like(x), torch.empty_like(x), pre=RMS)


def test_scales_as_tensors_are_read_at_the_call(cuda_dev):
    """A scale or an epsilon held in a tensor counts with the value that it has at the call."""
    x, y, *_ = _make(cuda_dev, 5, 64, torch.float16, torch.float16, torch.float16, 0)
    scale, eps = torch.tensor(1.0), torch.tensor(1e-5)
    for a, e in ((1.0, 1e-5), (0.25, 0.5), (-2.0, 4.0)):
        scale.fill_(a)
        eps.fill_(e)
        got = cuda_ext.block_norm(x, y, post=RMS, pre=LAYER, x_scale=scale, y_scale=scale, post_eps=eps, pre_eps=eps)
        want = cuda_ext.block_norm(x, y, post=RMS, pre=LAYER, x_scale=a, y_scale=a, post_eps=e, pre_eps=e)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
