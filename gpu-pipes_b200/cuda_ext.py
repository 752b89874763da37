"""Reference-compatible entry points: `cuda_ext.<app>(...)` and `cuda_ext.<app>_out(...)`.

The reference exposes each app as a pybind11 extension, e.g.
apps/mgn_fullmlp/pipelined/mgn_fullmlp_pl_ext.cu:24-93:
    mgn_fullmlp_out(x, w1, b1, w2, b2, w3, b3, gamma, beta, out) -> None
    mgn_fullmlp(x, w1, b1, w2, b2, w3, b3, gamma, beta) -> out
with weights in [K, N] layout (`linear.weight.t().contiguous()`, apps/mgn_fullmlp/pipelined/val.py:17-19).
The same names and argument meanings are kept here, so the reference's val.py / perf.py call
pattern (`ext.cuda_ext.mgn_fullmlp(...)`) works unchanged. Differences, all deliberate:
  * checks raise RuntimeError (the reference's TORCH_CHECK does too; its width `assert`s abort
    the process instead),
  * the launch goes to torch's current stream (the reference uses the legacy default stream),
  * M need not be a multiple of the reference's `n_rows * mblk`.
Each call goes through the C ABI (libgpipes.so) with raw device pointers.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib as L
from . import workloads as W

_DT = {torch.float16: L.GP_F16, torch.bfloat16: L.GP_BF16}


def _check_input(name: str, t: torch.Tensor | None, dtype: torch.dtype | None = None) -> None:
    if t is None:
        return
    if (type(t) is torch.Tensor and t.is_cuda and t.is_contiguous()
            and (dtype is None or t.dtype == dtype)):
        return  # the common case, in one test
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")


def _ptr(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(t: torch.Tensor) -> ctypes.c_void_p:
    """torch's current stream on t's device (the raw handle straight from torch's C layer where
    available: the Stream object costs a couple of microseconds per call)."""
    if _raw_stream is not None and t.device.index is not None:
        return ctypes.c_void_p(_raw_stream(t.device.index))
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


class _on_device:
    """`with torch.cuda.device(dev)`, skipped when `dev` is already current (the common case;
    switching costs microseconds of host time per call)."""

    __slots__ = ("idx", "prev")

    def __init__(self, dev: torch.device):
        self.idx = dev.index if dev.index is not None else torch.cuda.current_device()
        self.prev = None

    def __enter__(self):
        cur = torch.cuda.current_device()
        if cur != self.idx:
            self.prev = cur
            torch.cuda.set_device(self.idx)
        return self

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)
        return False


_SPECS: dict = {}


def _spec(widths, acts, tail, dt, ln_eps, skip_layer):
    """The chain description, built once per distinct chain (the struct is read-only to C)."""
    ln_eps = float(ln_eps)  # a tensor would be kept by its identity
    key = (tuple(widths), tuple(acts), tail, dt, ln_eps, skip_layer)
    s = _SPECS.get(key)
    if s is None:
        s = _SPECS[key] = L.make_spec(widths, acts, tail, dt, ln_eps, skip_layer)
    return s


def fused_mlp_out(x, weights, biases, out, *, acts, tail=L.TAIL_NONE, gamma=None, beta=None,
                  ln_eps=1e-5, skip_layer=0) -> None:
    """Generic chain: out = tail(act_L(... act_1(x W_1 + b_1) ...)). Weights are [K, N].

    skip_layer = s > 0: layer s reads [output of layer s-1 || x] and its weight is
    [N_{s-1} + K0, N_s] (the NeRF skip connection).

    weights may be W4Weight (all of them): the chain then runs on 4-bit weights (w4_mlp_out), which
    takes any widths and no skip layer."""
    for w in weights:
        if type(w) is W4Weight:
            if skip_layer:
                raise RuntimeError("skip_layer is not available on 4-bit weights")
            w4_mlp_out(x, weights, biases, out, acts=acts, tail=tail, gamma=gamma, beta=beta, ln_eps=ln_eps)
            return
    _check_input("x", x)
    dt = _DT.get(x.dtype)
    if dt is None:
        raise RuntimeError(f"x must be float16 or bfloat16, got {x.dtype}")
    for i, (w, b) in enumerate(zip(weights, biases)):
        _check_input(f"w{i + 1}", w, x.dtype)
        _check_input(f"b{i + 1}", b, x.dtype)
    _check_input("gamma", gamma, x.dtype)
    _check_input("beta", beta, x.dtype)
    _check_input("out", out, x.dtype)
    if x.dim() != 2 or out.dim() != 2:
        raise RuntimeError("x and out must be 2-D")
    widths = [x.shape[1]] + [w.shape[1] for w in weights]
    for i, w in enumerate(weights):
        k = widths[i] + (widths[0] if skip_layer and i == skip_layer else 0)
        if w.dim() != 2 or w.shape[0] != k:
            raise RuntimeError(f"w{i + 1} has shape {tuple(w.shape)}, expected [{k}, N]")
    if out.shape[0] != x.shape[0] or out.shape[1] != widths[-1]:
        raise RuntimeError(f"out has shape {tuple(out.shape)}, expected [{x.shape[0]}, {widths[-1]}]")
    spec = _spec(widths, acts, tail, dt, ln_eps, skip_layer)
    n = len(weights)
    wp = (ctypes.c_void_p * n)(*[w.data_ptr() for w in weights])
    bp = (ctypes.c_void_p * n)(*[(b.data_ptr() if b is not None else None) for b in biases])
    with _on_device(x.device):
        L.check(L.lib().gp_fused_mlp_out(ctypes.byref(spec), x.shape[0], _ptr(x), wp, bp,
                                         _ptr(gamma), _ptr(beta), _ptr(out), _stream(x)))


def fused_mlp_host_out(x_host, weights, biases, out_host, *, acts, tail=L.TAIL_NONE, gamma=None,
                       beta=None, ln_eps=1e-5, skip_layer=0, chunk_rows=0, device=None) -> None:
    """fused_mlp_out with x and out in HOST memory (pinned for overlap): the rows are streamed in
    chunks, H2D copies, kernels and D2H copies of neighbouring chunks overlapping. Weights and
    LayerNorm parameters are device tensors. Enqueued on the current stream of their device;
    synchronise it before reading out_host."""
    if x_host.is_cuda or out_host.is_cuda:
        raise RuntimeError("x_host and out_host must be host tensors")
    if not x_host.is_contiguous() or not out_host.is_contiguous():
        raise RuntimeError("x_host and out_host must be contiguous")
    dt = _DT.get(x_host.dtype)
    if dt is None or out_host.dtype != x_host.dtype:
        raise RuntimeError(f"x_host and out_host must both be float16 or bfloat16")
    dev = device if device is not None else weights[0].device
    for i, (w, b) in enumerate(zip(weights, biases)):
        _check_input(f"w{i + 1}", w, x_host.dtype)
        _check_input(f"b{i + 1}", b, x_host.dtype)
    _check_input("gamma", gamma, x_host.dtype)
    _check_input("beta", beta, x_host.dtype)
    widths = [x_host.shape[1]] + [w.shape[1] for w in weights]
    if out_host.dim() != 2 or out_host.shape[0] != x_host.shape[0] or out_host.shape[1] != widths[-1]:
        raise RuntimeError(f"out_host has shape {tuple(out_host.shape)}, expected [{x_host.shape[0]}, {widths[-1]}]")
    spec = L.make_spec(widths, acts, tail, dt, ln_eps, skip_layer)
    n = len(weights)
    wp = (ctypes.c_void_p * n)(*[w.data_ptr() for w in weights])
    bp = (ctypes.c_void_p * n)(*[(b.data_ptr() if b is not None else None) for b in biases])
    with torch.cuda.device(dev):
        L.check(L.lib().gp_fused_mlp_host(ctypes.byref(spec), x_host.shape[0],
                                          ctypes.c_void_p(x_host.data_ptr()), wp, bp, _ptr(gamma),
                                          _ptr(beta), ctypes.c_void_p(out_host.data_ptr()),
                                          int(chunk_rows),
                                          ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)))


# ------------------------------------------------------------------------------------------------
# MeshGraphNet family (apps/mgn_fullmlp, apps/mgn_linears, apps/test_mlp)
# ------------------------------------------------------------------------------------------------
def _mgn_checks(x, ws, bs, out, extra=()):
    _check_input("x", x, torch.float16)
    for i, (w, b) in enumerate(zip(ws, bs)):
        _check_input(f"w{i + 1}", w, torch.float16)
        _check_input(f"b{i + 1}", b, torch.float16)
    for name, t in extra:
        _check_input(name, t, torch.float16)
    _check_input("out", out, torch.float16)
    k0 = x.shape[1]
    shapes = [(k0, 128), (128, 128), (128, 128)]
    for i, (w, shp) in enumerate(zip(ws, shapes)):
        if tuple(w.shape) != shp:
            raise RuntimeError(f"w{i + 1} has shape {tuple(w.shape)}, expected {shp}")
    for i, b in enumerate(bs):
        if b is not None and tuple(b.shape) != (128,):
            raise RuntimeError(f"b{i + 1} has shape {tuple(b.shape)}, expected (128,)")
    if tuple(out.shape) != (x.shape[0], 128):
        raise RuntimeError(f"out has shape {tuple(out.shape)}, expected ({x.shape[0]}, 128)")


def mgn_fullmlp_out(x, w1, b1, w2, b2, w3, b3, gamma, beta, out) -> None:
    """x [M, K0] (K0 in 128/256/384) -> out [M, 128]; 3 Linear (ReLU, ReLU, none) + LayerNorm."""
    _mgn_checks(x, (w1, w2, w3), (b1, b2, b3), out, (("gamma", gamma), ("beta", beta)))
    with torch.cuda.device(x.device):
        L.check(L.lib().gp_mgn_fullmlp_out(x.shape[0], x.shape[1], _ptr(x), _ptr(w1), _ptr(b1),
                                           _ptr(w2), _ptr(b2), _ptr(w3), _ptr(b3), _ptr(gamma),
                                           _ptr(beta), _ptr(out), _stream(x)))


def mgn_fullmlp(x, w1, b1, w2, b2, w3, b3, gamma, beta) -> torch.Tensor:
    out = torch.zeros(x.shape[0], 128, dtype=x.dtype, device=x.device)
    mgn_fullmlp_out(x, w1, b1, w2, b2, w3, b3, gamma, beta, out)
    return out


def mgn_linears_out(x, w1, b1, w2, b2, w3, b3, out) -> None:
    _mgn_checks(x, (w1, w2, w3), (b1, b2, b3), out)
    with torch.cuda.device(x.device):
        L.check(L.lib().gp_mgn_linears_out(x.shape[0], x.shape[1], _ptr(x), _ptr(w1), _ptr(b1),
                                           _ptr(w2), _ptr(b2), _ptr(w3), _ptr(b3), _ptr(out),
                                           _stream(x)))


def mgn_linears(x, w1, b1, w2, b2, w3, b3) -> torch.Tensor:
    out = torch.zeros(x.shape[0], 128, dtype=x.dtype, device=x.device)
    mgn_linears_out(x, w1, b1, w2, b2, w3, b3, out)
    return out


def testmlp_out(x, w1, b1, w2, b2, w3, b3, out) -> None:
    if x.shape[1] != 128:
        raise RuntimeError(f"x has {x.shape[1]} columns, expected 128")
    _mgn_checks(x, (w1, w2, w3), (b1, b2, b3), out)
    with torch.cuda.device(x.device):
        L.check(L.lib().gp_testmlp_out(x.shape[0], _ptr(x), _ptr(w1), _ptr(b1), _ptr(w2),
                                       _ptr(b2), _ptr(w3), _ptr(b3), _ptr(out), _stream(x)))


def testmlp(x, w1, b1, w2, b2, w3, b3) -> torch.Tensor:
    out = torch.zeros(x.shape[0], 128, dtype=x.dtype, device=x.device)
    testmlp_out(x, w1, b1, w2, b2, w3, b3, out)
    return out


# ------------------------------------------------------------------------------------------------
# DLRM bottom MLP (apps/dlrm_botmlp), GraphCast MLPs (apps/gc_edges, apps/gc_nodes), NeRF
# ------------------------------------------------------------------------------------------------
def _out_like(x, n):
    return torch.zeros(x.shape[0], n, dtype=x.dtype, device=x.device)


def _check_chain(x, ws, bs, out, widths, dtype=torch.float16):
    """Shapes of a plain chain call: x [M, widths[0]], w_i [widths[i], widths[i+1]], b_i
    [widths[i+1]] (or None), out [M, widths[-1]]."""
    _check_input("x", x, dtype)
    _check_input("out", out, dtype)
    if x.dim() != 2 or x.shape[1] != widths[0]:
        raise RuntimeError(f"x has shape {tuple(x.shape)}, expected [M, {widths[0]}]")
    for i, (w, b) in enumerate(zip(ws, bs)):
        _check_input(f"w{i + 1}", w, dtype)
        _check_input(f"b{i + 1}", b, dtype)
        if w is None or tuple(w.shape) != (widths[i], widths[i + 1]):
            raise RuntimeError(f"w{i + 1} has shape {None if w is None else tuple(w.shape)}, "
                               f"expected {(widths[i], widths[i + 1])}")
        if b is not None and tuple(b.shape) != (widths[i + 1],):
            raise RuntimeError(f"b{i + 1} has shape {tuple(b.shape)}, expected ({widths[i + 1]},)")
    if out.dim() != 2 or tuple(out.shape) != (x.shape[0], widths[-1]):
        raise RuntimeError(f"out has shape {tuple(out.shape)}, expected [{x.shape[0]}, {widths[-1]}]")


def dlrm_botmlp_out(x, w1, b1, w2, b2, w3, b3, out) -> None:
    """x [M, K0] -> 512 -> 256 -> 128, ReLU after every layer. K0 = 32 is the reference app's own
    input (apps/dlrm_botmlp/pipelined/val.py:11-12, DlrmMlp([13 + 19, 512, 256, 128])); K0 = 16 is
    13 dense features zero padded (the benchmark config). Calls gp_dlrm_botmlp_out."""
    _check_input("x", x, torch.float16)
    k0 = x.shape[1] if x.dim() == 2 else -1
    _check_chain(x, [w1, w2, w3], [b1, b2, b3], out, [k0, 512, 256, 128])
    with torch.cuda.device(x.device):
        L.check(L.lib().gp_dlrm_botmlp_out(x.shape[0], k0, _ptr(x), _ptr(w1), _ptr(b1), _ptr(w2),
                                           _ptr(b2), _ptr(w3), _ptr(b3), _ptr(out), _stream(x)))


def dlrm_botmlp(x, w1, b1, w2, b2, w3, b3) -> torch.Tensor:
    out = _out_like(x, 128)
    dlrm_botmlp_out(x, w1, b1, w2, b2, w3, b3, out)
    return out


def gc_edges_out(x, w0, b0, w1, b1, ga, be, out, act=L.ACT_RELU) -> None:
    """x [M, 1536] -> 512 (act; ReLU as in the reference, SiLU for GraphCast) -> 512, LayerNorm."""
    fused_mlp_out(x, [w0, w1], [b0, b1], out, acts=[act, L.ACT_NONE], tail=L.TAIL_LAYERNORM,
                  gamma=ga, beta=be, ln_eps=1e-5)


def gc_edges(x, w0, b0, w1, b1, ga, be, act=L.ACT_RELU) -> torch.Tensor:
    out = _out_like(x, 512)
    gc_edges_out(x, w0, b0, w1, b1, ga, be, out, act=act)
    return out


gc_nodes_out = gc_edges_out  # x [M, 1024]; same chain shape after the first layer


def gc_nodes(x, w0, b0, w1, b1, ga, be, act=L.ACT_RELU) -> torch.Tensor:
    out = _out_like(x, 512)
    gc_nodes_out(x, w0, b0, w1, b1, ga, be, out, act=act)
    return out


def nerf_a_out(x, w1, b1, w2, b2, w3, b3, w4, b4, w5, b5, w6, b6, w7, b7, w8, b8, out) -> None:
    """NeRF trunk: x [M, 64] -> 256 (x5, ReLU), [h || x] -> 256 (w6 is [320, 256]), 256 x2."""
    fused_mlp_out(x, [w1, w2, w3, w4, w5, w6, w7, w8], [b1, b2, b3, b4, b5, b6, b7, b8], out,
                  acts=[L.ACT_RELU] * 8, skip_layer=5)


def nerf_a(x, *wb) -> torch.Tensor:
    out = _out_like(x, 256)
    nerf_a_out(x, *wb, out)
    return out


def nerf_out(x, weights, biases, out) -> None:
    """NeRF trunk + decode head 256 -> 4 (9 weights; the last one is [256, 4])."""
    fused_mlp_out(x, list(weights), list(biases), out, acts=[L.ACT_RELU] * 8 + [L.ACT_NONE],
                  skip_layer=5)


def _check_mgn_weights(k0, w1, b1, w2, b2, w3, b3, gamma, beta):
    for name, t, shape in (("w1", w1, (k0, 128)), ("w2", w2, (128, 128)), ("w3", w3, (128, 128)),
                           ("b1", b1, (128,)), ("b2", b2, (128,)), ("b3", b3, (128,)),
                           ("gamma", gamma, (128,)), ("beta", beta, (128,))):
        _check_input(name, t, torch.float16)
        if t is not None and tuple(t.shape) != shape:
            raise RuntimeError(f"{name} has shape {tuple(t.shape)}, expected {shape}")


def mgn_edge_update_out(nf, ef, srcs, dsts, w1, b1, w2, b2, w3, b3, gamma, beta, out,
                        agg=None) -> None:
    """MeshGraphNet edge update (graphmodel/mgn_dp.py:28-32) with the gather fused:
    out[e] = LN(MgnMlp([nf[srcs[e]] | ef[e] | nf[dsts[e]]])). nf [N, 128], ef [M, 128], srcs and
    dsts int64 [M], fp16. With agg (fp32 [N, 128]) the output rows are also summed into
    agg[dsts[e]] (accumulated onto agg's contents)."""
    _check_input("nf", nf, torch.float16)
    _check_input("ef", ef, torch.float16)
    _check_input("srcs", srcs, torch.int64)
    _check_input("dsts", dsts, torch.int64)
    _check_input("out", out, torch.float16)
    _check_input("agg", agg, torch.float32)
    m, n = ef.shape[0], nf.shape[0]
    if nf.dim() != 2 or nf.shape[1] != 128 or ef.dim() != 2 or ef.shape[1] != 128:
        raise RuntimeError(f"nf {tuple(nf.shape)} and ef {tuple(ef.shape)} must be [*, 128]")
    if tuple(srcs.shape) != (m,) or tuple(dsts.shape) != (m,):
        raise RuntimeError(f"srcs {tuple(srcs.shape)} and dsts {tuple(dsts.shape)} must be [{m}]")
    if tuple(out.shape) != (m, 128):
        raise RuntimeError(f"out has shape {tuple(out.shape)}, expected [{m}, 128]")
    if agg is not None and tuple(agg.shape) != (n, 128):
        raise RuntimeError(f"agg has shape {tuple(agg.shape)}, expected [{n}, 128]")
    _check_mgn_weights(384, w1, b1, w2, b2, w3, b3, gamma, beta)
    wp = (ctypes.c_void_p * 3)(w1.data_ptr(), w2.data_ptr(), w3.data_ptr())
    bp = (ctypes.c_void_p * 3)(*[None if t is None else t.data_ptr() for t in (b1, b2, b3)])
    with torch.cuda.device(ef.device):
        L.check(L.lib().gp_mgn_edge_update_out(m, n, _ptr(nf), _ptr(ef), _ptr(srcs), _ptr(dsts), wp,
                                               bp, _ptr(gamma), _ptr(beta), _ptr(out), _ptr(agg),
                                               _stream(ef)))


def mgn_edge_update(nf, ef, srcs, dsts, w1, b1, w2, b2, w3, b3, gamma, beta, agg=None):
    out = torch.empty(ef.shape[0], 128, dtype=ef.dtype, device=ef.device)
    mgn_edge_update_out(nf, ef, srcs, dsts, w1, b1, w2, b2, w3, b3, gamma, beta, out, agg=agg)
    return out


def mgn_node_update_out(nf, aggs, w1, b1, w2, b2, w3, b3, gamma, beta, out) -> None:
    """MeshGraphNet node update (graphmodel/mgn_dp.py:46-54): out = LN(MgnMlp([nf | aggs[0] |
    ...])), nf [N, 128] fp16, aggs: one or two fp32 [N, 128] edge-set aggregates (rounded to
    fp16 as the MLP input), w1 [128 (1 + len(aggs)), 128]."""
    aggs = list(aggs)
    _check_input("nf", nf, torch.float16)
    _check_input("out", out, torch.float16)
    n = nf.shape[0]
    if len(aggs) not in (1, 2):
        raise RuntimeError("one or two edge-set aggregates")
    for i, a in enumerate(aggs):
        _check_input(f"aggs[{i}]", a, torch.float32)
        if tuple(a.shape) != (n, 128):
            raise RuntimeError(f"aggs[{i}] has shape {tuple(a.shape)}, expected [{n}, 128]")
    if nf.dim() != 2 or nf.shape[1] != 128 or tuple(out.shape) != (n, 128):
        raise RuntimeError(f"nf {tuple(nf.shape)} and out {tuple(out.shape)} must be [{n}, 128]")
    _check_mgn_weights(128 * (1 + len(aggs)), w1, b1, w2, b2, w3, b3, gamma, beta)
    ap = (ctypes.c_void_p * 2)(*([a.data_ptr() for a in aggs] + [None] * (2 - len(aggs))))
    wp = (ctypes.c_void_p * 3)(w1.data_ptr(), w2.data_ptr(), w3.data_ptr())
    bp = (ctypes.c_void_p * 3)(*[None if t is None else t.data_ptr() for t in (b1, b2, b3)])
    with torch.cuda.device(nf.device):
        L.check(L.lib().gp_mgn_node_update_out(n, len(aggs), _ptr(nf), ap, wp, bp, _ptr(gamma),
                                               _ptr(beta), _ptr(out), _stream(nf)))


def mgn_node_update(nf, aggs, w1, b1, w2, b2, w3, b3, gamma, beta):
    out = torch.empty_like(nf)
    mgn_node_update_out(nf, aggs, w1, b1, w2, b2, w3, b3, gamma, beta, out)
    return out


_NERF_FULL_W = [(64, 256)] + [(256, 256)] * 4 + [(320, 256), (256, 256), (256, 256),
                (256, 64), (256, 256), (288, 128), (128, 64)]


def nerf_full_out(x, d, weights, biases, out_r, out_rgb) -> None:
    """NeRF with view directions (apps/nerf_full/pipelined/nerf_full_pl_ext.cu:22-95): x [M, 64],
    d [M, 32], weights w1..w12 ([K, N], shapes as the reference asserts), biases b1..b12 (entries
    may be None) -> out_r [M, 64] (alpha head), out_rgb [M, 64]. fp16."""
    _check_input("x", x, torch.float16)
    _check_input("d", d, torch.float16)
    _check_input("out_r", out_r, torch.float16)
    _check_input("out_rgb", out_rgb, torch.float16)
    m = x.shape[0]
    if x.dim() != 2 or x.shape[1] != 64:
        raise RuntimeError(f"x has shape {tuple(x.shape)}, expected [M, 64]")
    if tuple(d.shape) != (m, 32):
        raise RuntimeError(f"d has shape {tuple(d.shape)}, expected [{m}, 32]")
    for name, o in (("out_r", out_r), ("out_rgb", out_rgb)):
        if tuple(o.shape) != (m, 64):
            raise RuntimeError(f"{name} has shape {tuple(o.shape)}, expected [{m}, 64]")
    weights, biases = list(weights), list(biases) if biases is not None else [None] * 12
    if len(weights) != 12 or len(biases) != 12:
        raise RuntimeError("nerf_full takes 12 weights and 12 biases")
    for i, (wt, bt) in enumerate(zip(weights, biases)):
        _check_input(f"w{i + 1}", wt, torch.float16)
        _check_input(f"b{i + 1}", bt, torch.float16)
        if tuple(wt.shape) != _NERF_FULL_W[i]:
            raise RuntimeError(f"w{i + 1} has shape {tuple(wt.shape)}, expected {_NERF_FULL_W[i]}")
        if bt is not None and tuple(bt.shape) != (_NERF_FULL_W[i][1],):
            raise RuntimeError(f"b{i + 1} has shape {tuple(bt.shape)}, expected ({_NERF_FULL_W[i][1]},)")
    wp = (ctypes.c_void_p * 12)(*[wt.data_ptr() for wt in weights])
    bp = (ctypes.c_void_p * 12)(*[None if bt is None else bt.data_ptr() for bt in biases])
    with torch.cuda.device(x.device):
        L.check(L.lib().gp_nerf_full_out(m, _ptr(x), _ptr(d), wp, bp, _ptr(out_r), _ptr(out_rgb),
                                         _stream(x)))


def nerf_full(x, d, *wb):
    """nerf_full(x, d, w1, b1, ..., w12, b12) -> (out_r, out_rgb), like the reference's binding."""
    if len(wb) != 24:
        raise RuntimeError("nerf_full takes x, d and 12 (weight, bias) pairs")
    out_r = torch.zeros(x.shape[0], 64, dtype=x.dtype, device=x.device)
    out_rgb = torch.zeros_like(out_r)
    nerf_full_out(x, d, wb[0::2], wb[1::2], out_r, out_rgb)
    return out_r, out_rgb


def bert_ffn_out(x, w1, b1, w2, b2, ga, be, out, eps=None) -> None:
    """out = LN(x + W2 act(W1 x + b1) + b2).

    x [M, 128]: the reference's own BERT FFN (apps/bert_ffn: 128 -> 512 ReLU -> 128, LayerNorm eps
    1e-5), fp16 or bf16. x [M, 1024]: BERT-large (1024 -> 4096 GELU(tanh) -> 1024, eps 1e-12),
    bf16."""
    if x.dim() == 2 and x.shape[1] == 128:
        act0, eps = L.ACT_RELU, 1e-5 if eps is None else eps
    else:
        act0, eps = L.ACT_GELU_TANH, 1e-12 if eps is None else eps
    fused_mlp_out(x, [w1, w2], [b1, b2], out, acts=[act0, L.ACT_NONE],
                  tail=L.TAIL_RESIDUAL_LN, gamma=ga, beta=be, ln_eps=eps)


def bert_ffn(x, w1, b1, w2, b2, ga, be, eps=None) -> torch.Tensor:
    out = _out_like(x, x.shape[1])
    bert_ffn_out(x, w1, b1, w2, b2, ga, be, out, eps=eps)
    return out


def bert_addln_ffn_out(attn_out, x, w0, b0, w1, b1, w2, b2, ga0, be0, ga2, be2, out) -> None:
    """apps/bert_addln_ffn (H = 128, ff = 512, fp16): h = LN0(attn_out W0 + b0 + x),
    out = LN2(ReLU(h W1 + b1) W2 + b2 + h). Same argument order as the reference's
    bert_addln_ffn_out (bert_addln_ffn_pl_ext.cu:15-58)."""
    for name, t in (("attn_out", attn_out), ("x", x), ("out", out)):
        _check_input(name, t, torch.float16)
        if t.dim() != 2 or t.shape[1] != 128 or t.shape[0] != x.shape[0]:
            raise RuntimeError(f"{name} has shape {tuple(t.shape)}, expected [{x.shape[0]}, 128]")
    for name, w, shp in (("w0", w0, (128, 128)), ("w1", w1, (128, 512)), ("w2", w2, (512, 128))):
        _check_input(name, w, torch.float16)
        if tuple(w.shape) != shp:
            raise RuntimeError(f"{name} has shape {tuple(w.shape)}, expected {shp}")
    for name, t, n in (("b0", b0, 128), ("b1", b1, 512), ("b2", b2, 128), ("ga0", ga0, 128),
                       ("be0", be0, 128), ("ga2", ga2, 128), ("be2", be2, 128)):
        _check_input(name, t, torch.float16)
        if t is not None and tuple(t.shape) != (n,):
            raise RuntimeError(f"{name} has shape {tuple(t.shape)}, expected ({n},)")
    with torch.cuda.device(x.device):
        L.check(L.lib().gp_bert_addln_ffn_out(
            x.shape[0], _ptr(attn_out), _ptr(x), _ptr(w0), _ptr(b0), _ptr(w1), _ptr(b1), _ptr(w2),
            _ptr(b2), _ptr(ga0), _ptr(be0), _ptr(ga2), _ptr(be2), _ptr(out), _stream(x)))


def bert_addln_ffn(attn_out, x, w0, b0, w1, b1, w2, b2, ga0, be0, ga2, be2) -> torch.Tensor:
    """Allocating form. (The reference's passes be0 where be2 belongs,
    bert_addln_ffn_pl_ext.cu:74; this one passes be2.)"""
    out = _out_like(x, 128)
    bert_addln_ffn_out(attn_out, x, w0, b0, w1, b1, w2, b2, ga0, be0, ga2, be2, out)
    return out


def dlrm_interaction_out(bot, sparse, out) -> None:
    """DLRM feature interaction (graphmodel/dlrm.py:28-42): bot [M, 128] (bottom MLP output),
    sparse [M, 26, 128] (embedding vectors) -> out [M, 480] = [bot | 351 pairwise dot products
    below the diagonal, row-major | 0], the top MLP's input. fp16."""
    _check_input("bot", bot, torch.float16)
    _check_input("sparse", sparse, torch.float16)
    _check_input("out", out, torch.float16)
    m = bot.shape[0]
    if bot.dim() != 2 or bot.shape[1] != 128:
        raise RuntimeError(f"bot has shape {tuple(bot.shape)}, expected [M, 128]")
    if tuple(sparse.shape) != (m, 26, 128):
        raise RuntimeError(f"sparse has shape {tuple(sparse.shape)}, expected [{m}, 26, 128]")
    if tuple(out.shape) != (m, 480):
        raise RuntimeError(f"out has shape {tuple(out.shape)}, expected [{m}, 480]")
    with torch.cuda.device(bot.device):
        L.check(L.lib().gp_dlrm_interaction_out(m, _ptr(bot), _ptr(sparse), _ptr(out), _stream(bot)))


def dlrm_interaction(bot, sparse) -> torch.Tensor:
    out = torch.empty(bot.shape[0], 480, dtype=bot.dtype, device=bot.device)
    dlrm_interaction_out(bot, sparse, out)
    return out


def dlrm_topmlp_out(x, w1, b1, w2, b2, w3, b3, w4, b4, w5, b5, out) -> None:
    """Two width sets (gp_dlrm_topmlp_out):
      * x [M, 512] -> 1024 -> 1024 -> 512 -> 256 -> 64, ReLU after every layer: the reference
        app's own DlrmMlp([479 + 33, 1024, 1024, 512, 256, 64]) (apps/dlrm_topmlp/pipelined/val.py:11-12);
      * x [M, 480] -> 1024 -> 1024 -> 512 -> 256 (ReLU) -> 1 (sigmoid): DlrmMlp(..., sigmoid_i=4),
        the benchmark config."""
    _check_input("x", x, torch.float16)
    _check_input("w5", w5, torch.float16)
    k0 = x.shape[1] if x.dim() == 2 else -1
    n_out = w5.shape[1] if w5.dim() == 2 else -1
    ws, bs = [w1, w2, w3, w4, w5], [b1, b2, b3, b4, b5]
    _check_chain(x, ws, bs, out, [k0, 1024, 1024, 512, 256, n_out])
    wp = (ctypes.c_void_p * 5)(*[w.data_ptr() for w in ws])
    bp = (ctypes.c_void_p * 5)(*[(b.data_ptr() if b is not None else None) for b in bs])
    with torch.cuda.device(x.device):
        L.check(L.lib().gp_dlrm_topmlp_out(x.shape[0], k0, n_out, _ptr(x), wp, bp, _ptr(out),
                                           _stream(x)))


def dlrm_topmlp(x, *wb) -> torch.Tensor:
    out = _out_like(x, wb[8].shape[1])
    dlrm_topmlp_out(x, *wb, out)
    return out


# ------------------------------------------------------------------------------------------------
# Norms around a block, and layers with 4-bit weights (no reference counterpart)
# ------------------------------------------------------------------------------------------------
def _dtype_code(name, dtype):
    dt = _DT.get(dtype)
    if dt is None:
        raise RuntimeError(f"{name} must be float16 or bfloat16, got {dtype}")
    return dt


# These calls take microseconds on the GPU for single tokens, so their host side is kept short: one
# expression per tensor in the usual case (the messages are made in _refuse), raw addresses to ctypes.
_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _refuse(name, t, dtype, shape, dev) -> None:
    """Raise for a tensor that failed the short check (a non-tensor included)."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    _check_input(name, t, dtype)
    if tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.get_device() != dev:
        raise RuntimeError(f"{name} is on {t.device}, expected cuda:{dev}")
    raise RuntimeError(f"{name} cannot be used as {dtype} {tuple(shape)}")  # every refusal raises


def _address(name, t, dtype, shape, dev):
    """t's address if it is a contiguous tensor of that type and shape on CUDA device dev (an
    index); None for None."""
    if t is None:
        return None
    try:
        if t.dtype is dtype and t.get_device() == dev and t.shape == shape and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _refuse(name, t, dtype, shape, dev)
    return t.data_ptr()


def _cuda_2d(name, t):
    """The CUDA device index of a 2-D tensor."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise RuntimeError(f"{name} must be a 2-D tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _elsewhere(dev, fn, *args) -> int:
    """fn(*args, stream) with dev made the current device."""
    with _on_device(torch.device("cuda", dev)):
        return fn(*args, torch.cuda.current_stream(dev).cuda_stream)


def _launch(dev, fn, *args) -> None:
    """fn(*args, stream) on device dev's current stream, with dev as the current device."""
    if _raw_stream is not None and _get_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        rc = _elsewhere(dev, fn, *args)
    if rc != L.GP_OK:
        L.check(rc)


_NORM_SPECS: dict = {}


def _norm_spec(*key):
    s = _NORM_SPECS.get(key)
    if s is None:
        if len(_NORM_SPECS) >= 1024:  # gate_rows follows the row count: do not keep every one
            _NORM_SPECS.clear()
        s = _NORM_SPECS[key] = ctypes.byref(L.GpBlockNormSpec(*key))
    return s


def block_norm_out(x, y, r, h, *, post=L.NORM_NONE, pre=L.NORM_NONE, gate=None, post_gamma=None,
                   post_beta=None, pre_gamma=None, pre_beta=None, x_scale=1.0, y_scale=1.0,
                   post_eps=1e-5, pre_eps=1e-5) -> None:
    """Norms before and after a block with its gate and residual scales, one pass over the rows:

        r = x_scale x + y_scale gate * Npost(y),   h = Npre(r)

    N is L.NORM_NONE, L.NORM_LAYER or L.NORM_RMS (gamma and beta may be None). x [M, H] is the
    residual stream, y [M, H] the block's output; either may be None (without y: the norm before
    the first block; without x: no residual). gate: [H] for all rows, or [G, H] with M a multiple
    of G: one row for each M / G consecutive rows. r is the new stream, h the next block's input;
    either may be None. x and r have one type (16-bit, or float32 for a stream kept in 32 bits), y
    may be 16-bit or float32, h, gate, gammas and betas are float16 or bfloat16, all the same (float32
    ones are refused). r may be x or y and h may be x or y (in place) where the types match. Scales and
    epsilons are numbers; one held in a tensor is read at the call."""
    first = x if x is not None else y
    if first is None or (r is None and h is None):
        raise RuntimeError("block_norm needs x or y, and r or h")
    f32 = torch.float32
    dtype = None  # the 16-bit type of the call
    for t in (h, y, x, r, gate, post_gamma, post_beta, pre_gamma, pre_beta):
        if t is not None and getattr(t, "dtype", f32) is not f32:
            dtype = t.dtype
            break
    else:  # all fp32: only x, y and r may be
        for name, t in (("h", h), ("gate", gate), ("post_gamma", post_gamma), ("post_beta", post_beta),
                        ("pre_gamma", pre_gamma), ("pre_beta", pre_beta)):
            if t is not None:
                if not isinstance(t, torch.Tensor):
                    raise RuntimeError(f"{name} must be a tensor")
                raise RuntimeError(f"{name} must be float16 or bfloat16, got {t.dtype}")
    dev = _cuda_2d("x" if x is not None else "y", first)
    shape = first.shape
    m, width = shape
    dt = _DT.get(dtype) if dtype is not None else L.GP_F16  # all fp32: nothing is of that type
    if dt is None:
        _dtype_code("h", dtype)
    stream_t = x if x is not None else r
    stream = f32 if stream_t is not None and stream_t.dtype is f32 else dtype
    ydt = f32 if y is not None and y.dtype is f32 else dtype
    row = (width,)
    gate_rows, gate_shape = 0, row
    if gate is not None and getattr(gate, "ndim", 1) == 2:
        groups = gate.shape[0]
        if m and (groups == 0 or m % groups):
            raise RuntimeError(f"{m} rows are not a multiple of {groups} gate rows")
        gate_rows, gate_shape = m // groups if m else 0, (groups, width)
    _launch(dev, L.lib().gp_block_norm_out,
            _norm_spec(width, dt, stream is f32, ydt is f32, post, pre, float(post_eps), float(pre_eps), float(x_scale),
                       float(y_scale), gate_rows),
            m, None if x is None else _address("x", x, stream, shape, dev),
            None if y is None else _address("y", y, ydt, shape, dev),
            None if gate is None else _address("gate", gate, dtype, gate_shape, dev),
            None if post_gamma is None else _address("post_gamma", post_gamma, dtype, row, dev),
            None if post_beta is None else _address("post_beta", post_beta, dtype, row, dev),
            None if pre_gamma is None else _address("pre_gamma", pre_gamma, dtype, row, dev),
            None if pre_beta is None else _address("pre_beta", pre_beta, dtype, row, dev),
            None if r is None else _address("r", r, stream, shape, dev),
            None if h is None else _address("h", h, dtype, shape, dev))


def block_norm(x, y=None, *, dtype=None, want_r=True, post=L.NORM_NONE, pre=L.NORM_NONE, **kw):
    """block_norm_out with new outputs: (r, h). r is None without y or with want_r=False, h is None
    without a norm before the next block. dtype: h's type where x and y are both float32 (float16
    or bfloat16; default the type of y, x or the parameters)."""
    first = x if x is not None else y
    if first is None:
        raise RuntimeError("block_norm needs x or y")
    r = h = None
    if want_r and y is not None:
        r = torch.empty_like(first)
    if pre != L.NORM_NONE:
        if dtype is None:
            for t in (y, x, *kw.values()):
                if isinstance(t, torch.Tensor) and t.dtype in _DT:
                    dtype = t.dtype
                    break
            else:
                raise RuntimeError("dtype must be given where every tensor is float32")
        h = torch.empty_like(first) if first.dtype is dtype else torch.empty_like(first, dtype=dtype)
    block_norm_out(x, y, r, h, post=post, pre=pre, **kw)
    return r, h


@functools.lru_cache(maxsize=1024)
def _w4_spec(k, n, group, dtype, zero_points):
    """(the C description, bytes of the packed form)"""
    spec = ctypes.byref(L.GpW4Spec(k, n, group, _dtype_code("weights", dtype), int(zero_points)))
    nbytes = L.lib().gp_w4_packed_bytes(spec)
    if nbytes < 0:
        L.check(int(nbytes))
    return spec, nbytes


class W4Weight:
    """Weights [K, N] in 4 bits with group scales along K (gp_w4_spec): the packed buffer and what
    it holds. Made by w4_quantize or w4_pack."""

    __slots__ = ("packed", "k", "n", "group", "dtype", "zero_points", "spec", "nbytes")

    def __init__(self, packed, k, n, group, dtype, zero_points):
        self.k, self.n, self.group = int(k), int(n), int(group)
        self.dtype, self.zero_points = dtype, bool(zero_points)
        self.spec, self.nbytes = _w4_spec(self.k, self.n, self.group, dtype, self.zero_points)
        if packed is not None:
            _check_input("packed", packed, torch.uint8)
            if tuple(packed.shape) != (self.nbytes,):
                raise RuntimeError(f"packed has shape {tuple(packed.shape)}, expected ({self.nbytes},)")
        self.packed = packed

    @classmethod
    def empty(cls, k, n, group, dtype, zero_points, device):
        """An unfilled weight on `device`."""
        w = cls(None, k, n, group, dtype, zero_points)
        w.packed = torch.empty(w.nbytes, dtype=torch.uint8, device=device)
        return w

    @property
    def shape(self):
        return (self.k, self.n)

    @property
    def device(self):
        return self.packed.device

    def _address(self, name, dev):
        return _address(name, self.packed, torch.uint8, (self.nbytes,), dev)

    def _unpack(self, rows, dtype, place):
        t = torch.empty(rows, self.n, dtype=dtype, device=self.device)
        outs = [None, None, None]
        outs[place] = t.data_ptr()
        dev = self.packed.get_device()
        _launch(dev, L.lib().gp_w4_unpack_out, self.spec, self._address("packed", dev), *outs)
        return t

    def codes(self):
        """q [K, N], one code (0..15) per byte."""
        return self._unpack(self.k, torch.uint8, 0)

    def scales(self):
        """s [ceil(K / group), N]."""
        return self._unpack(-(-self.k // self.group), self.dtype, 1)

    def zeros(self):
        """z [ceil(K / group), N] (bytes 0..15), or None without zero points."""
        return self._unpack(-(-self.k // self.group), torch.uint8, 2) if self.zero_points else None


def w4_quantize_out(w, w4) -> None:
    """Quantise w [K, N] (float16 or bfloat16) into a W4Weight of the same shape and type."""
    dev = _cuda_2d("w", w)
    _launch(dev, L.lib().gp_w4_quantize_out, w4.spec, _address("w", w, w4.dtype, (w4.k, w4.n), dev),
            w4._address("packed", dev))


def w4_quantize(w, group=128, zero_points=False) -> W4Weight:
    """w [K, N] to 4 bits: per group of `group` rows and column, the largest magnitude becomes code
    distance 7 (or, with zero_points, the range with zero becomes 0..15); gp_w4_quantize_out has
    the rule."""
    dev = _cuda_2d("w", w)
    w4 = W4Weight.empty(w.shape[0], w.shape[1], group, w.dtype, zero_points, w.device)
    w4_quantize_out(w, w4)
    return w4


def w4_pack(codes, scales, zeros=None, group=128) -> W4Weight:
    """Weights quantised elsewhere: codes uint8 [K, N] (0..15), scales [ceil(K / group), N] (float16
    or bfloat16, the type of the activations), zeros uint8 of the scales' shape or None (8)."""
    dev = _cuda_2d("codes", codes)
    _cuda_2d("scales", scales)
    k, n = codes.shape
    w4 = W4Weight.empty(k, n, group, scales.dtype, zeros is not None, codes.device)
    rows = (-(-k // group), n)
    _launch(dev, L.lib().gp_w4_pack_out, w4.spec, _address("codes", codes, torch.uint8, (k, n), dev),
            _address("scales", scales, scales.dtype, rows, dev),
            _address("zeros", zeros, torch.uint8, rows, dev), w4.packed.data_ptr())
    return w4


def w4_dequantize_out(w4, w) -> None:
    """w [K, N] = s (q - z), rounded once."""
    dev = _cuda_2d("w", w)
    _launch(dev, L.lib().gp_w4_dequantize_out, w4.spec, w4._address("packed", dev),
            _address("w", w, w4.dtype, (w4.k, w4.n), dev))


def w4_dequantize(w4) -> torch.Tensor:
    w = torch.empty(w4.k, w4.n, dtype=w4.dtype, device=w4.device)
    w4_dequantize_out(w4, w)
    return w


def w4_linear_out(x, w4, bias, out, act=L.ACT_NONE) -> None:
    """out [M, N] = act(x [M, K] W + bias) on 4-bit weights; x, bias (or None) and out have the
    weights' type. Single tokens, decode batches, prompts. From 17 rows on each weight is rounded to 16
    bits first; w4_mlp_out of the one layer rounds none."""
    if not isinstance(w4, W4Weight):
        raise RuntimeError("w4 must be a W4Weight")
    dev = _cuda_2d("x", x)
    m, dtype = x.shape[0], w4.dtype
    if out is None:
        raise RuntimeError("out must be a tensor")
    _launch(dev, L.lib().gp_w4_linear_out, w4.spec, m, act, _address("x", x, dtype, (m, w4.k), dev),
            w4._address("packed", dev), _address("bias", bias, dtype, (w4.n,), dev),
            _address("out", out, dtype, (m, w4.n), dev))


def w4_linear(x, w4, bias=None, act=L.ACT_NONE) -> torch.Tensor:
    if not isinstance(w4, W4Weight):
        raise RuntimeError("w4 must be a W4Weight")
    out = torch.empty(x.shape[0], w4.n, dtype=x.dtype, device=x.device)
    w4_linear_out(x, w4, bias, out, act=act)
    return out


@functools.lru_cache(maxsize=None)
def _pointer_array(n):
    return ctypes.c_void_p * n


_W4_CHAINS: dict = {}


def _w4_chain(m, widths, acts, tail, dtype, ln_eps):
    """The chain's description and the workspace bytes of m rows."""
    ln_eps = float(ln_eps)  # a tensor would be kept by its identity
    key = (m, widths, acts, tail, dtype, ln_eps)
    c = _W4_CHAINS.get(key)
    if c is None:
        spec = L.make_spec(widths, acts, tail, _DT[dtype], ln_eps, 0)
        nbytes = L.lib().gp_w4_mlp_workspace_bytes(ctypes.byref(spec), m)
        if nbytes < 0:
            L.check(int(nbytes))
        if len(_W4_CHAINS) >= 1024:
            _W4_CHAINS.clear()
        c = _W4_CHAINS[key] = (ctypes.byref(spec), int(nbytes))
    return c


def w4_mlp_out(x, weights, biases, out, *, acts, tail=L.TAIL_NONE, gamma=None, beta=None,
               ln_eps=1e-5, workspace=None) -> None:
    """The generic chain of fused_mlp_out on 4-bit weights (a list of W4Weight of one group size,
    type and kind of zero points): any widths, every activation and tail. workspace: a uint8 CUDA
    tensor of at least w4_mlp_workspace_bytes; None takes one from torch's allocator. out may be x
    where the chain has a tail and ends in x's width."""
    n = len(weights)
    if n == 0 or len(biases) != n or len(acts) != n:
        raise RuntimeError(f"{n} weights, {len(biases)} biases and {len(acts)} activations must match")
    for w in weights:
        if not isinstance(w, W4Weight):
            raise RuntimeError("either every weight of a chain is a W4Weight, or none")
    dev = _cuda_2d("x", x)
    w0 = weights[0]
    dtype, m, width = w0.dtype, x.shape[0], w0.k
    xp = _address("x", x, dtype, (m, width), dev)
    wp, bp, widths = [], [], [width]
    for i in range(n):
        w = weights[i]
        if w.group != w0.group or w.dtype != dtype or w.zero_points != w0.zero_points:
            raise RuntimeError(f"w{i + 1} differs from w1 in group size, type or zero points")
        if w.k != width:
            raise RuntimeError(f"w{i + 1} has shape {w.shape}, expected [{width}, N]")
        width = w.n
        widths.append(width)
        wp.append(w._address("w", dev))
        bp.append(_address("bias", biases[i], dtype, (width,), dev))
    gp, ep = _address("gamma", gamma, dtype, (width,), dev), _address("beta", beta, dtype, (width,), dev)
    if out is None:
        raise RuntimeError("out must be a tensor")
    op = _address("out", out, dtype, (m, width), dev)
    spec, nbytes = _w4_chain(m, tuple(widths), tuple(acts), tail, dtype, ln_eps)
    if workspace is None:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    else:
        _address("workspace", workspace, torch.uint8, (workspace.numel(),), dev)
    ptrs = _pointer_array(n)
    _launch(dev, L.lib().gp_w4_mlp_out, spec, w0.group, int(w0.zero_points), m, xp, ptrs(*wp), ptrs(*bp), gp, ep,
            op, None if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.numel())


def w4_mlp_workspace_bytes(m, weights, *, acts, tail=L.TAIL_NONE) -> int:
    """Workspace of a w4_mlp_out call on m rows."""
    widths = (weights[0].k,) + tuple(w.n for w in weights)
    return _w4_chain(m, widths, tuple(acts), tail, weights[0].dtype, 1e-5)[1]


def w4_mlp(x, weights, biases, *, acts, tail=L.TAIL_NONE, gamma=None, beta=None, ln_eps=1e-5) -> torch.Tensor:
    out = torch.empty(x.shape[0], weights[-1].n, dtype=x.dtype, device=x.device)
    w4_mlp_out(x, weights, biases, out, acts=acts, tail=tail, gamma=gamma, beta=beta, ln_eps=ln_eps)
    return out


def run_workload_host(w, x_host, weights, ln, out_host) -> None:
    """A plain-chain workloads.Workload end to end on host buffers (gp_fused_mlp_host)."""
    if w.block:
        raise RuntimeError(f"{w.name}: host pipeline covers plain chains only")
    gamma, beta = ln if ln is not None else (None, None)
    fused_mlp_host_out(x_host, [p[0] for p in weights], [p[1] for p in weights], out_host,
                       acts=w.acts, tail=w.tail, gamma=gamma, beta=beta, ln_eps=w.ln_eps,
                       skip_layer=w.skip_layer)


_SCRATCH = {}


def _scratch_f32(device, n):
    """A cached fp32 device buffer of at least n elements per device (grown, never shrunk)."""
    key = (device.type, device.index)
    buf = _SCRATCH.get(key)
    if buf is None or buf.numel() < n:
        buf = torch.empty(n, dtype=torch.float32, device=device)
        _SCRATCH[key] = buf
    return buf[:n]


def run_workload_out(w, x, weights, ln, out) -> None:
    """Run a workloads.Workload chain through the generic C entry point."""
    if w.block == "dlrm_interaction":
        m = x.shape[0] // 27
        dlrm_interaction_out(x[:m], x[m:].view(m, 26, x.shape[1]), out)
        return
    if w.block == "mgn_mp":
        ef, nf, srcs, dsts = W.split_mgn_input(x)
        m, n = ef.shape[0], nf.shape[0]
        o = out.view(-1)
        agg = _scratch_f32(x.device, n * 128).view(n, 128)
        agg.zero_()
        (e1, e2, e3, n1, n2, n3) = weights
        ge, be, gn, bn = ln
        mgn_edge_update_out(nf, ef, srcs, dsts, e1[0], e1[1], e2[0], e2[1], e3[0], e3[1], ge, be,
                            o[:m * 128].view(m, 128), agg=agg)
        mgn_node_update_out(nf, [agg], n1[0], n1[1], n2[0], n2[1], n3[0], n3[1], gn, bn,
                            o[m * 128:].view(n, 128))
        return
    if w.block == "nerf_full":
        m = x.numel() // 96
        o = out.view(-1)
        nerf_full_out(x[:m * 64].view(m, 64), x[m * 64:].view(m, 32), [p[0] for p in weights],
                      [p[1] for p in weights], o[:m * 64].view(m, 64), o[m * 64:].view(m, 64))
        return
    if w.block == "bert_addln":
        m = x.shape[0] // 2
        (w0, b0), (w1, b1), (w2, b2) = weights
        ga0, be0, ga2, be2 = ln
        bert_addln_ffn_out(x[:m], x[m:], w0, b0, w1, b1, w2, b2, ga0, be0, ga2, be2, out)
        return
    gamma, beta = ln if ln is not None else (None, None)
    fused_mlp_out(x, [p[0] for p in weights], [p[1] for p in weights], out, acts=w.acts,
                  tail=w.tail, gamma=gamma, beta=beta, ln_eps=w.ln_eps, skip_layer=w.skip_layer)
