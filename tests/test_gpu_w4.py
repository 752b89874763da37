"""4-bit weights on the GPU: quantising, packing and reading back against the rule in 64 bits,
products and chains against the products of the codes in 64 bits."""
import math

import pytest
import torch

from gpu_pipes_b200 import _lib as L
from gpu_pipes_b200 import cuda_ext
from tests._tol import U32, check, half_step, rounded, tiny

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


# ------------------------------------------------------------------------------------------------
# references
# ------------------------------------------------------------------------------------------------
def quantize_ref(w, group, zeros):
    """(codes, scales, zero points) by the documented rule, in 64 bits."""
    k, n = w.shape
    ng = -(-k // group)
    codes = torch.zeros(k, n, dtype=torch.uint8)
    scales = torch.zeros(ng, n, dtype=w.dtype)
    zs = torch.zeros(ng, n, dtype=torch.uint8)
    for g in range(ng):
        part = w[g * group:(g + 1) * group].double()
        lo, hi = part.amin(0).clamp(max=0), part.amax(0).clamp(min=0)
        s = ((hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7).to(w.dtype)
        sd = s.double()
        safe = torch.where(sd > 0, sd, 1.0)
        z = torch.round(-lo / safe).clamp(0, 15) * (sd > 0) if zeros else torch.full_like(sd, 8.0)
        q = torch.round(part / safe) + z
        q = torch.where(sd > 0, q, z).clamp(0, 15)
        codes[g * group:(g + 1) * group] = q.to(torch.uint8)
        scales[g] = s
        zs[g] = z.to(torch.uint8)
    return codes, scales, zs if zeros else None


def weights64(codes, scales, zeros, group):
    k = codes.shape[0]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 0)[:k]
    return (codes.double() - z) * scales.double().repeat_interleave(group, 0)[:k]


def act64(a, v):
    if a == L.ACT_RELU:
        return v.clamp(min=0)
    if a == L.ACT_GELU_TANH:
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if a == L.ACT_SILU:
        return v * torch.sigmoid(v)
    if a == L.ACT_SIGMOID:
        return torch.sigmoid(v)
    return v


def linear_ref(x, xerr, w, bias, act, dtype):
    """(act(x w + b), error bound before a store) for x within xerr. The sums: products of 16-bit
    values are exact in fp32; the matrix unit adds 16 at a time and may truncate, at most a step
    (2 U32) of the magnitudes per addition, K / 16 of them if none were independent, then at most
    64 + 16 + 8 joins. More than 16 rows go to the kernel that rounds each weight to T, at most half a
    step of it. An activation has slope at most 1.13 and costs a few half steps, tanh's
    cancellation among them (relative to |v|, not to the result)."""
    k = w.shape[0]
    v = x @ w
    mag = x.abs() @ w.abs()
    err = xerr @ w.abs() + 2 * U32 * (k / 16 + 96) * mag
    if x.shape[0] > 16:
        err = err + half_step(dtype) * (mag + xerr @ w.abs()) + tiny(dtype) * x.abs().sum(1, keepdim=True)
    if bias is not None:
        v, err = v + bias.double(), err + U32 * (v.abs() + bias.double().abs())
    if act not in (L.ACT_NONE, L.ACT_RELU):
        err = 1.13 * err + 16 * U32 * (v.abs() + 1)
    return act64(act, v), err


def make(k, n, dtype, group, zeros, seed=0, dev="cuda:0"):
    """Random codes over all 16 values, scales and zero points."""
    g = torch.Generator().manual_seed(seed * 1009 + k * 31 + n)
    ng = -(-k // group)
    codes = torch.randint(0, 16, (k, n), generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(ng, n, generator=g)) / (4 * math.sqrt(k))).to(dtype)
    z = torch.randint(0, 16, (ng, n), generator=g, dtype=torch.uint8) if zeros else None
    return codes.to(dev), scales.to(dev), None if z is None else z.to(dev)


def rows(m, k, dtype, seed=1, dev="cuda:0"):
    g = torch.Generator().manual_seed(seed * 7 + m * 13 + k)
    return torch.randn(m, k, generator=g).to(dtype).to(dev)


# ------------------------------------------------------------------------------------------------
# quantising and packing
# ------------------------------------------------------------------------------------------------
SHAPES = [(8, 1), (64, 16), (72, 17), (128, 40), (200, 33), (1000, 130), (1024, 514), (4104, 96)]


@pytest.mark.parametrize("k,n", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize(cuda_dev, k, n, group, zeros):
    for dtype in DTYPES:
        g = torch.Generator().manual_seed(k + n)
        w = (torch.randn(k, n, generator=g) * torch.exp(torch.randn(n, generator=g))).to(dtype)
        w[: k // 2, n // 2] = 0  # groups of zeros
        w4 = cuda_ext.w4_quantize(w.to(cuda_dev), group=group, zero_points=zeros)
        codes, scales, z = quantize_ref(w, group, zeros)
        assert torch.equal(w4.codes().cpu(), codes)
        assert torch.equal(w4.scales().cpu(), scales)
        assert (w4.zeros() is None) == (z is None)
        if zeros:
            assert torch.equal(w4.zeros().cpu(), z)
        deq = cuda_ext.w4_dequantize(w4).cpu()
        assert torch.equal(deq, weights64(codes, scales, z, group).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_ties_and_extremes(cuda_dev, dtype):
    """Values exactly between two codes (half to even), the largest finite values, subnormal
    groups, one-sided groups, and groups that are not finite."""
    k, n = 64, 16
    w = torch.zeros(k, n, dtype=dtype)
    s = 2.0 ** -3
    w[:15, 0] = torch.tensor([(i - 7) * s for i in range(15)]).to(dtype)  # every code
    w[15:29, 0] = torch.tensor([(i - 6.5) * s for i in range(14)]).to(dtype)  # every tie
    w[:, 1] = 7 * s * 3
    w[:28, 1] = torch.tensor([(i - 13.5) * 0.5 * s * 3 for i in range(28)]).to(dtype)
    big = 6e4 if dtype == torch.float16 else 1e38
    w[:, 2] = torch.linspace(-big, big, k).to(dtype) * (1 if dtype == torch.bfloat16 else 0.5)
    w[:, 3] = torch.tensor(2.0 ** -22).to(dtype) * torch.arange(k)  # fp16: subnormal
    w[5, 4] = 2.0 ** -24  # fp16: a scale that rounds to zero
    w[:, 5] = torch.rand(k, generator=torch.Generator().manual_seed(1)).to(dtype) + 1  # positive
    w[:, 6] = -w[:, 5]
    for zeros in (False, True):
        w4 = cuda_ext.w4_quantize(w.to(cuda_dev), group=64, zero_points=zeros)
        codes, scales, z = quantize_ref(w, 64, zeros)
        assert torch.equal(w4.scales().cpu(), scales)
        assert torch.equal(w4.codes().cpu(), codes)
        if zeros:
            assert torch.equal(w4.zeros().cpu(), z)
        bad = w.clone()
        bad[3, 9], bad[4, 10], bad[5, 11] = float("nan"), float("inf"), -float("inf")
        b4 = cuda_ext.w4_quantize(bad.to(cuda_dev), group=64, zero_points=zeros)
        sc = b4.scales().cpu()
        assert not sc[0, 9:12].isfinite().any()
        keep = [c for c in range(n) if c not in (9, 10, 11)]
        assert torch.equal(sc[:, keep], scales[:, keep])
        assert torch.equal(b4.codes().cpu()[:, keep], codes[:, keep])
        assert not cuda_ext.w4_dequantize(b4).cpu()[:, 9:12].isfinite().any()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n", [24, 23])
def test_quantize_smallest_bf16_groups(cuda_dev, n, zeros):
    """Groups down to bf16's smallest numbers: 1 / s is past fp32's range for s of 2^-128 and less. Each
    column is whole numbers (zeros and both signs among them) times 2^(c - 133)."""
    g = torch.Generator().manual_seed(n)
    ints = torch.randint(-120, 121, (160, n), generator=g).double()
    ints[3], ints[7] = 0, 120
    ints[64:128, 1] = torch.arange(64).double() % 4 - 2  # a scale that rounds to zero or to the smallest number
    ints[64:128, 2] = torch.arange(64).double() % 12 - 1
    w = (ints * torch.pow(2.0, torch.arange(n).double() - 133)).to(torch.bfloat16)
    assert torch.equal(w.double(), ints * torch.pow(2.0, torch.arange(n).double() - 133))
    for group in (32, 64, 128):
        w4 = cuda_ext.w4_quantize(w.to(cuda_dev), group=group, zero_points=zeros)
        codes, scales, z = quantize_ref(w, group, zeros)
        assert torch.equal(w4.scales().cpu(), scales)
        assert torch.equal(w4.codes().cpu(), codes)
        if zeros:
            assert torch.equal(w4.zeros().cpu(), z)


@pytest.mark.parametrize("n", [8, 7])
def test_quantize_widest_bf16_range(cuda_dev, n):
    """Groups whose range hi - lo is past fp32's largest number, (hi - lo) / 15 well within it."""
    big = torch.finfo(torch.bfloat16).max
    w = torch.linspace(-1, 1, 72 * n, dtype=torch.float64).view(72, n) * 3e38
    w[0], w[1] = big, -big
    w[2:4, 1] = torch.tensor([1.8e38, -1.75e38], dtype=torch.float64)
    w = w.to(torch.bfloat16)
    for group in (32, 64, 128):
        w4 = cuda_ext.w4_quantize(w.to(cuda_dev), group=group, zero_points=True)
        codes, scales, z = quantize_ref(w, group, True)
        assert scales.isfinite().all()
        assert torch.equal(w4.scales().cpu(), scales)
        assert torch.equal(w4.codes().cpu(), codes)
        assert torch.equal(w4.zeros().cpu(), z)
    w[5, 0], w[6, 1], w[7, 2] = float("inf"), -float("inf"), float("nan")
    sc = cuda_ext.w4_quantize(w.to(cuda_dev), group=128, zero_points=True).scales().cpu()
    assert not sc[:, :3].isfinite().any() and sc[:, 3:].isfinite().all()


@pytest.mark.parametrize("k,n", SHAPES)
@pytest.mark.parametrize("zeros", [False, True])
def test_pack_round_trip(cuda_dev, k, n, zeros):
    for group in (32, 64, 128):
        for dtype in DTYPES:
            codes, scales, z = make(k, n, dtype, group, zeros)
            w4 = cuda_ext.w4_pack(codes, scales, z, group=group)
            assert torch.equal(w4.codes(), codes)
            assert torch.equal(w4.scales(), scales)
            if zeros:
                assert torch.equal(w4.zeros(), z)
            want = weights64(codes, scales, z, group).to(dtype)
            assert torch.equal(cuda_ext.w4_dequantize(w4), want)


def test_unaligned_views(cuda_dev):
    """Matrices that start on a 2-byte boundary, and one whose width is odd."""
    dtype, k, n = torch.float16, 72, 34
    flat = torch.randn(k * n + 1, generator=torch.Generator().manual_seed(3)).to(dtype).to(cuda_dev)
    w = flat[1:].view(k, n)
    a, b = cuda_ext.w4_quantize(w, group=32), cuda_ext.w4_quantize(w.clone(), group=32)
    assert torch.equal(a.packed, b.packed)
    out = torch.zeros(k * n + 2, dtype=dtype, device=cuda_dev)
    cuda_ext.w4_dequantize_out(a, out[1:-1].view(k, n))
    assert torch.equal(out[1:-1].view(k, n), cuda_ext.w4_dequantize(b))
    assert out[0] == 0 and out[-1] == 0


# ------------------------------------------------------------------------------------------------
# products
# ------------------------------------------------------------------------------------------------
def check_linear(m, k, n, dtype, group, zeros, act, bias, dev, seed=0):
    codes, scales, z = make(k, n, dtype, group, zeros, seed)
    x = rows(m, k, dtype)
    b = rows(1, n, dtype, 5)[0].contiguous() if bias else None
    w4 = cuda_ext.w4_pack(codes, scales, z, group=group)
    buf = torch.full((m + 2, n), 7.0, dtype=dtype, device=dev)
    cuda_ext.w4_linear_out(x, w4, b, buf[:m], act=act)
    ref, err = linear_ref(x.double(), torch.zeros_like(x, dtype=torch.float64), weights64(codes, scales, z, group), b, act, dtype)
    check(buf[:m], ref, rounded(ref, err, dtype), f"{m}x{k}x{n}")
    assert (buf[m:] == 7).all()  # rows behind the last stay


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 15, 16, 17, 33, 64, 100, 129, 300])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_rows(cuda_dev, m, zeros):
    for dtype in DTYPES:
        check_linear(m, 1096, 520, dtype, 64, zeros, L.ACT_NONE, True, cuda_dev)


@pytest.mark.parametrize("k,n", [(8, 1), (8, 300), (32, 16), (64, 15), (72, 4), (120, 2368), (1024, 4096), (4096, 1024),
                                 (4104, 77), (5128, 1003), (9224, 40), (16384, 48), (28680, 24), (65536, 16),
                                 (64, 40000)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_linear_shapes(cuda_dev, k, n, group):
    for m, dtype, zeros in ((1, torch.float16, True), (3, torch.bfloat16, False), (16, torch.float16, False),
                            (40, torch.bfloat16, True)):
        check_linear(m, k, n, dtype, group, zeros, L.ACT_NONE, False, cuda_dev)


@pytest.mark.parametrize("m", [17, 128, 129, 257, 530])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_tiles(cuda_dev, m, group, zeros):
    """Row tiles of every kind of the kernel for more rows: one and two accumulators, two and four
    dequantising groups, several tiles, absent column tiles, K alone and split over a cluster."""
    for k, n in ((328, 264), (2056, 136)):
        check_linear(m, k, n, torch.float16 if zeros else torch.bfloat16, group, zeros, L.ACT_SILU, True, cuda_dev)


@pytest.mark.parametrize("act", [L.ACT_NONE, L.ACT_RELU, L.ACT_GELU_TANH, L.ACT_SILU, L.ACT_SIGMOID])
@pytest.mark.parametrize("m", [1, 20, 200])
def test_linear_activations(cuda_dev, act, m):
    for dtype in DTYPES:
        check_linear(m, 256, 272, dtype, 128, False, act, True, cuda_dev)


def test_linear_many_rows(cuda_dev):
    check_linear(20001, 64, 24, torch.float16, 32, True, L.ACT_RELU, True, cuda_dev)


def test_linear_large_offsets(cuda_dev):
    """Packed codes past 2^31 bytes from the buffer's start: the last columns of a very wide layer."""
    k, n, m = 32768, 140000, 2
    w4 = cuda_ext.W4Weight.empty(k, n, 128, torch.bfloat16, False, cuda_dev)
    assert w4.packed.numel() > 2**31
    w4.packed.zero_()  # code 0, scale 0 ...
    tail = 48
    codes, scales, _ = make(k, tail, torch.bfloat16, 128, False)
    t4 = cuda_ext.w4_pack(codes, scales, None, group=128)
    cells = k // 128  # of a 16-column tile: 1,024 bytes of codes each, then 32 of scales
    at, so, to = (n - tail) // 16 * cells, n // 16 * cells * 1024, tail // 16 * cells * 1024
    w4.packed[at * 1024:so] = t4.packed[:to]
    w4.packed[so + at * 32:] = t4.packed[to:]
    x = rows(m, k, torch.bfloat16)
    out = cuda_ext.w4_linear(x, w4)
    assert torch.equal(out[:, -tail:], cuda_ext.w4_linear(x, t4))
    assert (out[:, :-tail] == 0).all()


def test_linear_infinities_stay_in_their_row_and_column(cuda_dev):
    for m in (4, 40, 150):
        codes, scales, z = make(256, 96, torch.float16, 64, False)
        x = rows(m, 256, torch.float16)
        w4 = cuda_ext.w4_pack(codes, scales, None, group=64)
        clean = cuda_ext.w4_linear(x, w4)
        x2 = x.clone()
        x2[1, 5] = float("nan")
        x2[3, 255] = float("inf")
        out = cuda_ext.w4_linear(x2, w4)
        keep = [i for i in range(m) if i not in (1, 3)]
        assert torch.equal(out[keep], clean[keep])
        assert out[1].isnan().all() and not out[3].isfinite().any()
        s2 = scales.clone()
        s2[2, 17] = float("nan")
        out = cuda_ext.w4_linear(x, cuda_ext.w4_pack(codes, s2, None, group=64))
        cols = [i for i in range(96) if i != 17]
        assert torch.equal(out[:, cols], clean[:, cols]) and out[:, 17].isnan().all()


@pytest.mark.parametrize("m", [1, 3, 8, 9, 16, 17, 70])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_outliers_that_meet_zero_weights(cuda_dev, m, zeros):
    """Values of x far above the rest whose weights are all zero (q = z) take nothing from the others'
    sums, in a layer and in a chain: the bound has |x| |w| in it, not |x| and the codes."""
    for dtype, big in ((torch.bfloat16, 2.0 ** 30), (torch.float16, 6e4)):
        for group in (32, 128):
            k, n = 1096, 200
            codes, scales, z = make(k, n, dtype, group, zeros)
            hot = torch.arange(5, k, 61, device=codes.device)
            codes[hot] = torch.full_like(codes[hot], 8) if z is None else z[hot // group]
            x = rows(m, k, dtype)
            x[:, hot] = big
            w4 = cuda_ext.w4_pack(codes, scales, z, group=group)
            ref, err = linear_ref(x.double(), torch.zeros_like(x, dtype=torch.float64),
                                  weights64(codes, scales, z, group), None, L.ACT_NONE, dtype)
            if m > 16:  # tiny weights' rounding, here of weights that are not tiny
                err = err - tiny(dtype) * x.double().abs().sum(1, keepdim=True)
            check(cuda_ext.w4_linear(x, w4), ref, rounded(ref, err, dtype), f"m={m} {dtype}")
            check(cuda_ext.w4_mlp(x, [w4], [None], acts=[L.ACT_NONE]), ref, rounded(ref, err, dtype), f"chain m={m} {dtype}")


@pytest.mark.parametrize("m", [2, 8, 16, 20])
def test_linear_infinite_rows_follow_the_definition(cuda_dev, m):
    """An infinite x gives plus or minus infinity, or NaN where it meets a weight of zero or the other
    infinity, at any number of rows. Large finite values stay finite where their products with q - z do
    (64 times 2^119 times 24 would not)."""
    for dtype in DTYPES:
        for zeros in (False, True):
            codes, scales, z = make(256, 96, dtype, 64, zeros)
            x = rows(m, 256, dtype)
            x[0, 5] = float("inf")
            x[1, 250] = -float("inf")
            w = weights64(codes, scales, z, 64)
            got, ref = cuda_ext.w4_linear(x, cuda_ext.w4_pack(codes, scales, z, group=64)).double(), x.double() @ w
            assert torch.equal(got[:2].nan_to_num(7.0, 1.0, -1.0), ref[:2].nan_to_num(7.0, 1.0, -1.0))
            assert got[2:].isfinite().all()
    x = rows(m, 256, torch.bfloat16)
    x[0, :128] = 2.0 ** 119
    codes, scales, z = make(256, 96, torch.bfloat16, 64, False)
    scales = (scales.double() * 2.0 ** -100).to(torch.bfloat16)
    ref, err = linear_ref(x.double(), torch.zeros_like(x, dtype=torch.float64), weights64(codes, scales, z, 64), None,
                          L.ACT_NONE, torch.bfloat16)
    check(cuda_ext.w4_linear(x, cuda_ext.w4_pack(codes, scales, z, group=64)), ref, rounded(ref, err, torch.bfloat16), f"m={m}")


def test_linear_is_repeatable(cuda_dev):
    for m in (1, 12, 64):
        codes, scales, z = make(4096, 2000, torch.bfloat16, 128, True)
        w4 = cuda_ext.w4_pack(codes, scales, z, group=128)
        x = rows(m, 4096, torch.bfloat16)
        first = cuda_ext.w4_linear(x, w4)
        for _ in range(5):
            assert torch.equal(cuda_ext.w4_linear(x, w4), first)


def test_linear_misaligned_out_and_bias(cuda_dev):
    dtype = torch.float16
    for m in (3, 50):
        codes, scales, _ = make(128, 33, dtype, 64, False)
        w4 = cuda_ext.w4_pack(codes, scales, None, group=64)
        x = rows(m, 128, dtype)
        bias = rows(1, 34, dtype)[0]
        want = cuda_ext.w4_linear(x, w4, bias[1:].clone())
        flat = torch.full((m * 33 + 2,), 7.0, dtype=dtype, device=cuda_dev)
        cuda_ext.w4_linear_out(x, w4, bias[1:], flat[1:-1].view(m, 33))
        assert torch.equal(flat[1:-1].view(m, 33), want)
        assert flat[0] == 7 and flat[-1] == 7


# ------------------------------------------------------------------------------------------------
# chains
# ------------------------------------------------------------------------------------------------
def mlp_ref(x, layers, biases, acts, tail, gamma, beta, eps, group, dtype):
    v, err = x.double(), torch.zeros_like(x, dtype=torch.float64)
    for i, (codes, scales, z) in enumerate(layers):
        last = i + 1 == len(layers)
        act = L.ACT_NONE if last and tail else acts[i]
        v, err = linear_ref(v, err, weights64(codes, scales, z, group), biases[i], act, dtype)
        if not last:
            err = rounded(v, err, dtype)  # hidden activations are stored in 16 bits
    if not tail:
        return v, rounded(v, err, dtype)
    if tail == L.TAIL_RESIDUAL_LN:
        err = err + U32 * (v.abs() + x.double().abs())
        v = v + x.double()
    c = 128 * U32  # as the block norms' tests derive it
    d = v - v.mean(1, keepdim=True)
    e = err + err.mean(1, keepdim=True) + c * (v.abs() + 2 * v.abs().mean(1, keepdim=True))
    rs = 1 / torch.sqrt(d.square().mean(1, keepdim=True) + eps)
    rel = 2 * torch.sqrt(e.square().mean(1, keepdim=True)) * rs + c
    n = d * rs * gamma.double()
    out = n + beta.double()
    return out, rounded(out, e * rs * gamma.double().abs() + n.abs() * rel + c * (n.abs() + beta.double().abs()), dtype)


CHAINS = [((64, 64), (0,), 0), ((128, 200, 24), (1, 0), 0), ((128, 512, 128), (1, 0), 2),
          ((1024, 4096, 1024), (2, 0), 2), ((256, 136, 72, 264), (3, 4, 0), 1), ((72, 80, 88, 96, 7), (1, 2, 3, 4), 0),
          ((8, 8), (0,), 2)]


@pytest.mark.parametrize("widths,acts,tail", CHAINS)
@pytest.mark.parametrize("m", [1, 5, 37, 130])
def test_mlp(cuda_dev, widths, acts, tail, m):
    for dtype, group, zeros in ((torch.bfloat16, 128, False), (torch.float16, 32, True)):
        layers = [make(k, n, dtype, group, zeros, i) for i, (k, n) in enumerate(zip(widths[:-1], widths[1:]))]
        ws = [cuda_ext.w4_pack(*layer, group=group) for layer in layers]
        biases = [None if i == 1 else rows(1, n, dtype, 9)[0].contiguous() for i, n in enumerate(widths[1:])]
        x = rows(m, widths[0], dtype)
        gamma = (rows(1, widths[-1], dtype, 3)[0] * 0.1 + 1).contiguous() if tail else None
        beta = rows(1, widths[-1], dtype, 4)[0].contiguous() if tail else None
        out = torch.full((m + 1, widths[-1]), 7.0, dtype=dtype, device=cuda_dev)
        before = L.launch_count()
        cuda_ext.fused_mlp_out(x, ws, biases, out[:m], acts=list(acts), tail=tail, gamma=gamma, beta=beta, ln_eps=1e-5)
        assert L.launch_count() >= before + len(ws) + (1 if tail else 0)
        ref, bound = mlp_ref(x, layers, biases, acts, tail, gamma, beta, 1e-5, group, dtype)
        check(out[:m], ref, bound, f"{widths} m={m}")
        assert (out[m] == 7).all()
        got = cuda_ext.w4_mlp(x, ws, biases, acts=list(acts), tail=tail, gamma=gamma, beta=beta, ln_eps=1e-5)
        assert torch.equal(got, out[:m])
        if tail == L.TAIL_RESIDUAL_LN:  # in place
            y = x.clone()
            cuda_ext.w4_mlp_out(y, ws, biases, y, acts=list(acts), tail=tail, gamma=gamma, beta=beta, ln_eps=1e-5)
            assert torch.equal(y, got)


@pytest.mark.parametrize("m", [7, 16, 33])
def test_mlp_wide_hidden_layer(cuda_dev, m):
    """A hidden layer so wide that the rows of the next product, two T per value, take more than one pass."""
    widths, dtype, group = (64, 40008, 24, 8), torch.float16, 128
    layers = [make(k, n, dtype, group, True, i) for i, (k, n) in enumerate(zip(widths[:-1], widths[1:]))]
    ws = [cuda_ext.w4_pack(*layer, group=group) for layer in layers]
    x, acts = rows(m, widths[0], dtype), [L.ACT_SILU, L.ACT_GELU_TANH, L.ACT_NONE]
    got = cuda_ext.w4_mlp(x, ws, [None] * 3, acts=acts)
    ref, bound = mlp_ref(x, layers, [None] * 3, acts, 0, None, None, 1e-5, group, dtype)
    check(got, ref, bound, f"m={m}")


@pytest.mark.parametrize("widths", [(128, 512, 128), (256, 136, 72, 264), (72, 80, 88, 96, 40)])
@pytest.mark.parametrize("m", [9, 37, 130])
def test_roundings_of_a_chain(cuda_dev, widths, m):
    """What a chain's result is off by, as a root mean square, against the rounding of the exact result.
    No weight is rounded and longer chains keep their hidden activations as two T: what is left is the
    final rounding. Two layers round the hidden activations once: independent relative errors of the
    terms of a sum are at most as much of the sum, so sqrt(2) of the final rounding in all. Both with a
    tenth for the sample (360 values or more: the root mean square of as many roundings varies by 2.4%),
    and fp32's sums and the products of second parts on top, within their bounds."""
    for dtype, group, zeros in ((torch.bfloat16, 128, False), (torch.float16, 32, True)):
        layers = [make(k, n, dtype, group, zeros, i) for i, (k, n) in enumerate(zip(widths[:-1], widths[1:]))]
        ws = [cuda_ext.w4_pack(*layer, group=group) for layer in layers]
        x = rows(m, widths[0], dtype)
        got = cuda_ext.w4_mlp(x, ws, [None] * len(ws), acts=[L.ACT_RELU] * (len(ws) - 1) + [L.ACT_NONE]).double()
        v, err = x.double(), torch.zeros_like(x, dtype=torch.float64)
        for i, (codes, scales, z) in enumerate(layers):
            w = weights64(codes, scales, z, group)
            mag = v.abs() @ w.abs()
            # up to three products per term, and the parts left out
            err = err @ w.abs() + (2 * U32 * (3 * w.shape[0] / 16 + 96) + 2 * half_step(dtype) ** 2) * mag
            v = v @ w
            if i + 1 < len(layers):
                v = v.clamp(min=0)
        rms = lambda t: t.square().mean().sqrt().item()  # noqa: E731
        final = rms(v.to(dtype).double() - v)
        assert rms(got - v) <= 1.1 * final * (2 ** 0.5 if len(layers) == 2 else 1.0) + rms(err), (widths, m, dtype)


@pytest.mark.parametrize("tail", [L.TAIL_NONE, L.TAIL_LAYERNORM, L.TAIL_RESIDUAL_LN])
@pytest.mark.parametrize("m", [9, 17, 37, 130])
def test_roundings_of_a_chain_of_one_layer(cuda_dev, m, tail):
    """One layer through the chain's entry point rounds no weight either: what is left is the final
    rounding. As in test_roundings_of_a_chain, with a tenth for the sample (4,600 values or more); before a
    tail the sum stays in fp32, and the norm's arithmetic is as mlp_ref derives it, without the term for
    rounded weights that it has above 16 rows."""
    k = 512
    for dtype, group, zeros in ((torch.bfloat16, 128, False), (torch.float16, 32, True), (torch.bfloat16, 32, True)):
        layer = make(k, k, dtype, group, zeros, 3)
        w = weights64(*layer, group)
        x = rows(m, k, dtype)
        got = cuda_ext.w4_mlp(x, [cuda_ext.w4_pack(*layer, group=group)], [None], acts=[L.ACT_NONE], tail=tail)
        v, x = x.double() @ w, x.double()
        err = 2 * U32 * (2 * k / 16 + 96) * (x.abs() @ w.abs())
        if tail:
            c = 128 * U32
            v = v + (x if tail == L.TAIL_RESIDUAL_LN else 0)
            e = err + err.mean(1, keepdim=True) + c * (v.abs() + x.abs() + 2 * v.abs().mean(1, keepdim=True))
            d = v - v.mean(1, keepdim=True)
            rs = 1 / torch.sqrt(d.square().mean(1, keepdim=True) + 1e-5)
            v = d * rs
            err = e * rs + v.abs() * (2 * torch.sqrt(e.square().mean(1, keepdim=True)) * rs + c)
        rms = lambda t: t.square().mean().sqrt().item()  # noqa: E731
        assert rms(got.double() - v) <= 1.1 * rms(v.to(dtype).double() - v) + rms(err), (m, tail, dtype)


@pytest.mark.parametrize("act", [L.ACT_SILU, L.ACT_GELU_TANH, L.ACT_SIGMOID])
@pytest.mark.parametrize("tail", [L.TAIL_NONE, L.TAIL_RESIDUAL_LN])
@pytest.mark.parametrize("m", [12, 33, 140])
def test_roundings_of_a_chain_with_activations_and_tails(cuda_dev, act, tail, m):
    """test_roundings_of_a_chain with activations, biases and tails (3,168 values or more): the residual,
    the biases and the norm only add to what the errors are measured against."""
    for dtype, group, zeros in ((torch.bfloat16, 64, True), (torch.bfloat16, 128, False), (torch.float16, 128, False)):
        for widths in ((264, 520, 264), (264, 136, 392, 264)):
            layers = [make(k, n, dtype, group, zeros, i) for i, (k, n) in enumerate(zip(widths[:-1], widths[1:]))]
            ws = [cuda_ext.w4_pack(*layer, group=group) for layer in layers]
            biases = [rows(1, n, dtype, 9)[0].contiguous() for n in widths[1:]]
            x, nl = rows(m, widths[0], dtype), len(layers)
            got = cuda_ext.w4_mlp(x, ws, biases, acts=[act] * (nl - 1) + [L.ACT_NONE], tail=tail)
            v, err, x = x.double(), torch.zeros_like(x, dtype=torch.float64), x.double()
            for i, layer in enumerate(layers):
                w = weights64(*layer, group)
                mag = v.abs() @ w.abs()
                err = err @ w.abs() + (2 * U32 * (3 * w.shape[0] / 16 + 96) + 2 * half_step(dtype) ** 2) * mag
                v = v @ w + biases[i].double()
                err = err + U32 * (v.abs() + biases[i].double().abs())
                if i + 1 < nl:
                    err, v = 1.13 * err + 16 * U32 * (v.abs() + 1), act64(act, v)
            if tail:
                c = 128 * U32
                v = v + x
                e = err + err.mean(1, keepdim=True) + c * (v.abs() + x.abs() + 2 * v.abs().mean(1, keepdim=True))
                d = v - v.mean(1, keepdim=True)
                rs = 1 / torch.sqrt(d.square().mean(1, keepdim=True) + 1e-5)
                v = d * rs
                err = e * rs + v.abs() * (2 * torch.sqrt(e.square().mean(1, keepdim=True)) * rs + c)
            rms = lambda t: t.square().mean().sqrt().item()  # noqa: E731
            final = rms(v.to(dtype).double() - v)
            assert rms(got.double() - v) <= 1.1 * final * (2 ** 0.5 if nl == 2 else 1.0) + rms(err), (widths, m, dtype)


@pytest.mark.parametrize("m", [5, 16, 17, 40, 150])
@pytest.mark.parametrize("layers", [1, 2, 3])
def test_chain_with_fp16_weights_past_the_largest_number(cuda_dev, m, layers):
    """s (q - z) past 65,504 with scales that are finite: the sum is finite at any number of rows. The
    first layer's weights are quantised ones (the largest fp16 number becomes 7 x 9,360 = 65,520, which
    rounds to infinity) or packed ones up to 8 x 16,000; its products are small enough for the hidden
    values to be finite. Past 65,504 the second of a weight's two parts is at most 65,504, so what its
    rounding takes is at most 16: half_step times the weight, relative to at least 65,504."""
    dtype, group = torch.float16, 64
    g = torch.Generator().manual_seed(m)
    k, n = 136, 72
    big = (torch.randn(k, n, generator=g) * 2e4).clamp(-65504, 65504)
    big[::9] = 65504.0 * torch.sign(big[::9])
    w4 = cuda_ext.w4_quantize(big.to(dtype).to(cuda_dev), group=group)
    quantised = (w4.codes(), w4.scales(), None)
    assert weights64(*quantised, group).abs().max() > 65504
    codes, scales, _ = make(k, n, dtype, group, False)
    packed = (codes, (scales.float() / scales.float().max() * 16000).to(dtype), None)
    rest = [make(72, 72, dtype, group, False, i) for i in range(1, layers)]
    acts = [L.ACT_RELU] * (layers - 1) + [L.ACT_NONE]
    x = (rows(m, k, dtype).double() * 2.0 ** -12).to(dtype)
    for first in (quantised, packed):
        chain = [first, *rest]
        ws = [cuda_ext.w4_pack(*layer, group=group) for layer in chain]
        got = cuda_ext.w4_mlp(x, ws, [None] * layers, acts=acts)
        ref, bound = mlp_ref(x, chain, [None] * layers, acts, 0, None, None, 1e-5, group, dtype)
        assert got.isfinite().all()
        check(got, ref, bound, f"m={m}")
        if first is quantised and layers == 1:  # every such weight is two fp16 numbers: exact
            final = (ref.to(dtype).double() - ref).square().mean().sqrt()
            sums = 2 * U32 * (3 * k / 16 + 96) * (x.double().abs() @ weights64(*first, group).abs())
            assert (got.double() - ref).square().mean().sqrt() <= 1.1 * final + sums.square().mean().sqrt()


def test_chain_epsilon_as_a_tensor_is_read_at_the_call(cuda_dev):
    w4 = cuda_ext.w4_pack(*make(64, 64, torch.float16, 64, False), group=64)
    x, eps = rows(3, 64, torch.float16), torch.tensor(1e-5)
    for e in (1e-5, 0.5, 8.0):
        eps.fill_(e)
        kw = dict(acts=[L.ACT_NONE], tail=L.TAIL_LAYERNORM)
        assert torch.equal(cuda_ext.w4_mlp(x, [w4], [None], ln_eps=eps, **kw), cuda_ext.w4_mlp(x, [w4], [None], ln_eps=e, **kw))


def test_bert_ffn_takes_packed_weights(cuda_dev):
    """The BERT-large block's entry point with 4-bit weights, against the same block on the 16-bit
    values that they stand for: the fused 16-bit chain has its own roundings (fp16 hidden
    activations, tanh approximation), so both are held to the repository's parity tolerance."""
    from oracle import mlp_oracle as O
    dtype = torch.bfloat16
    g = torch.Generator().manual_seed(2)
    w1 = cuda_ext.w4_quantize((torch.randn(1024, 4096, generator=g) * 0.02).to(dtype).to(cuda_dev))
    w2 = cuda_ext.w4_quantize((torch.randn(4096, 1024, generator=g) * 0.02).to(dtype).to(cuda_dev))
    x = rows(24, 1024, dtype)
    one, zero = torch.ones(1024, dtype=dtype, device=cuda_dev), torch.zeros(1024, dtype=dtype, device=cuda_dev)
    out = cuda_ext.bert_ffn(x, w1, None, w2, None, one, zero)
    full = cuda_ext.bert_ffn(x, cuda_ext.w4_dequantize(w1), None, cuda_ext.w4_dequantize(w2), None, one, zero)
    r = O.compare(out.float().cpu(), full.float().cpu())
    assert r["max_abs"] <= 2 * O.MAX_ABS_TOL and r["rel_l2"] <= O.REL_L2_TOL, r


# ------------------------------------------------------------------------------------------------
# a run of them together
# ------------------------------------------------------------------------------------------------
def _block(dev, dtype, h=768, f=1544, layers=3, group=64):
    """A pre-norm feed-forward stack for serving: packed weights and norm parameters."""
    out = []
    for i in range(layers):
        up, down = make(h, f, dtype, group, False, 2 * i), make(f, h, dtype, group, False, 2 * i + 1)
        out.append(dict(up=cuda_ext.w4_pack(*up, group=group), down=cuda_ext.w4_pack(*down, group=group),
                        gamma=(rows(1, h, dtype, 20 + i)[0] * 0.1 + 1).contiguous(),
                        post=(rows(1, h, dtype, 40 + i)[0] * 0.1 + 1).contiguous(),
                        gate=(rows(1, h, dtype, 60 + i)[0] * 0.1 + 0.5).contiguous()))
    return out


def _serve(x, blocks, sync=False):
    """x through the stack: norm, up (SiLU), down, norm + gate + residual + next norm."""
    wait = torch.cuda.synchronize if sync else (lambda: None)
    _, h = cuda_ext.block_norm(x, pre=L.NORM_RMS, pre_gamma=blocks[0]["gamma"])
    r = x
    for i, b in enumerate(blocks):
        wait()
        u = cuda_ext.w4_linear(h, b["up"], act=L.ACT_SILU)
        wait()
        d = cuda_ext.w4_linear(u, b["down"])
        wait()
        nxt = blocks[i + 1]["gamma"] if i + 1 < len(blocks) else None
        r, h = cuda_ext.block_norm(r, d, post=L.NORM_RMS, post_gamma=b["post"], gate=b["gate"], y_scale=0.5,
                                   pre=L.NORM_RMS if nxt is not None else L.NORM_NONE, pre_gamma=nxt)
    wait()
    return r


@pytest.mark.parametrize("m", [1, 11, 70])
def test_stack_without_waiting_equals_stack_with(cuda_dev, m):
    """Launches overlap (programmatic dependent launch); every buffer here is the next call's
    input, so a read before its writer has finished would show."""
    for dtype in DTYPES:
        blocks = _block(cuda_dev, dtype)
        x = rows(m, 768, dtype)
        want = _serve(x, blocks, sync=True)
        for _ in range(10):
            assert torch.equal(_serve(x, blocks), want)


@pytest.mark.parametrize("m", [1, 70])
def test_two_graphs_share_nothing(cuda_dev, m):
    """Captured without an eager call before, replayed on new inputs, two graphs at a time on two
    streams: no workspace joins them."""
    dtype = torch.float16
    blocks = _block(cuda_dev, dtype)
    gamma = torch.ones(768, dtype=dtype, device=cuda_dev)
    beta = torch.zeros_like(gamma)

    def step(x):
        r = _serve(x, blocks)
        return cuda_ext.w4_mlp(r, [blocks[0]["up"], blocks[0]["down"]], [None, None], acts=[L.ACT_SILU, 0],
                               tail=L.TAIL_RESIDUAL_LN, gamma=gamma, beta=beta)

    xs = [rows(m, 768, dtype, 70 + i) for i in range(4)]
    bufs = [torch.empty_like(xs[0]) for _ in range(2)]
    graphs, outs = [], []
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(b))
        graphs.append(g)
    wants = [step(x) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, j in ((0, 1), (2, 3), (3, 0)):
        bufs[0].copy_(xs[i])
        bufs[1].copy_(xs[j])
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], wants[i]) and torch.equal(outs[1], wants[j])


def test_weights_written_just_before(cuda_dev):
    """Quantise into one buffer again and again, each followed by a product on it, unsynchronised."""
    dtype = torch.bfloat16
    ws = [rows(512, 640, dtype, 80 + i) for i in range(4)]
    x = rows(3, 512, dtype)
    want = [cuda_ext.w4_linear(x, cuda_ext.w4_quantize(w)) for w in ws]
    torch.cuda.synchronize()
    w4 = cuda_ext.W4Weight.empty(512, 640, 128, dtype, False, cuda_dev)
    got = []
    for _ in range(3):
        for w in ws:
            cuda_ext.w4_quantize_out(w, w4)
            got.append(cuda_ext.w4_linear(x, w4))
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 4])


def test_chain_kernels_next_to_them(cuda_dev):
    """A 16-bit chain reads what a block norm or a packed layer has just written, and the other way
    round, unsynchronised: the launch overlap's records cover both."""
    dtype = torch.float16
    g = torch.Generator().manual_seed(4)
    w = [(torch.randn(128, 128, generator=g) * 0.1).to(dtype).to(cuda_dev) for _ in range(3)]
    b = [torch.zeros(128, dtype=dtype, device=cuda_dev) for _ in range(3)]
    w4 = cuda_ext.w4_pack(*make(128, 128, dtype, 64, False), group=64)
    x0 = rows(5000, 128, dtype)

    def run(sync):
        wait = torch.cuda.synchronize if sync else (lambda: None)
        x = x0.clone()
        h = torch.empty_like(x)
        for _ in range(4):
            cuda_ext.block_norm_out(x, None, None, h, pre=L.NORM_LAYER)
            wait()
            cuda_ext.testmlp_out(h, w[0], b[0], w[1], b[1], w[2], b[2], x)
            wait()
            cuda_ext.w4_linear_out(x, w4, None, h)
            wait()
            cuda_ext.testmlp_out(h, w[0], b[0], w[1], b[1], w[2], b[2], x)
            wait()
        torch.cuda.synchronize()
        return x

    want = run(True)
    for _ in range(5):
        assert torch.equal(run(False), want)


def test_host_threads(cuda_dev):
    """Calls of several host threads at once, each on its own stream and buffers."""
    import threading

    dtype = torch.float16
    w4 = cuda_ext.w4_pack(*make(1024, 520, dtype, 64, True), group=64)
    xs = [rows(m, 1024, dtype, m) for m in (1, 5, 16, 40)]
    wants = [cuda_ext.w4_linear(x, w4) for x in xs]
    norms = [cuda_ext.block_norm(x, x, pre=L.NORM_RMS)[1] for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got, h = cuda_ext.w4_linear(xs[i], w4), cuda_ext.block_norm(xs[i], xs[i], pre=L.NORM_RMS)[1]
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(got, wants[i]) and torch.equal(h, norms[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one():
    for m in (2, 40):
        codes, scales, z = make(256, 96, torch.float16, 64, True, dev="cuda:1")
        x = rows(m, 256, torch.float16, dev="cuda:1")
        got = cuda_ext.w4_linear(x, cuda_ext.w4_pack(codes, scales, z, group=64))
        _, h = cuda_ext.block_norm(x, pre=L.NORM_RMS)
        assert got.device == h.device == x.device
        w4 = cuda_ext.w4_pack(codes.to("cuda:0"), scales.to("cuda:0"), z.to("cuda:0"), group=64)
        assert torch.equal(got.to("cuda:0"), cuda_ext.w4_linear(x.to("cuda:0"), w4))


def test_device_refusals(cuda_dev):
    dtype = torch.float16
    w4 = cuda_ext.w4_pack(*make(64, 32, dtype, 64, False), group=64)
    x = rows(2, 64, dtype)
    with pytest.raises(RuntimeError, match="must be torch.float16"):
        cuda_ext.w4_linear(x.bfloat16(), w4)
    with pytest.raises(RuntimeError, match=r"expected \(2, 64\)"):
        cuda_ext.w4_linear(x[:, :32].contiguous(), w4)
    with pytest.raises(RuntimeError, match="bias"):
        cuda_ext.w4_linear(x, w4, x[0])
    with pytest.raises(L.GpError, match="16-byte"):
        cuda_ext.w4_linear(torch.zeros(2 * 64 + 4, dtype=dtype, device=cuda_dev)[4:].view(2, 64), w4)
    with pytest.raises(RuntimeError, match="scales"):
        cuda_ext.w4_pack(torch.zeros(64, 32, dtype=torch.uint8, device=cuda_dev),
                         torch.zeros(2, 32, dtype=dtype, device=cuda_dev), group=64)
    with pytest.raises(L.GpError, match="workspace"):
        cuda_ext.w4_mlp_out(x, [w4], [None], torch.empty(2, 32, dtype=dtype, device=cuda_dev), acts=[0],
                            tail=L.TAIL_LAYERNORM, workspace=torch.empty(16, dtype=torch.uint8, device=cuda_dev))
    with pytest.raises(RuntimeError, match="differs"):
        other = cuda_ext.w4_pack(*make(32, 32, dtype, 32, False), group=32)
        cuda_ext.w4_mlp(x, [w4, other], [None, None], acts=[0, 0])
    empty = cuda_ext.w4_linear(x[:0], w4)
    assert empty.shape == (0, 32)


def test_missing_codes_time_out_and_the_next_call_is_right(cuda_dev):
    """With host-side fault injection no block of codes is ever loaded: every wait runs out after
    5 ms, the kernel ends, the status word says so, and the context stays usable."""
    for m, k, n in ((1, 256, 64), (8, 16384, 48), (40, 256, 2000), (40, 4096, 48)):  # both kernels, alone and in clusters
        codes, scales, z = make(k, n, torch.float16, 64, True)
        w4 = cuda_ext.w4_pack(codes, scales, z, group=64)
        x = rows(m, k, torch.float16)
        want = cuda_ext.w4_linear(x, w4)
        assert L.device_status(0, clear=True) == 0
        try:
            L.set_timeout_ns(5_000_000)
            L.set_fault_injection(1)
            cuda_ext.w4_linear(x, w4)
            torch.cuda.synchronize()
        finally:
            L.set_fault_injection(0)
            L.set_timeout_ns(0)
        assert L.device_status(0, clear=True) in (0x100, 0x200, 0x300)  # whichever role gave up first
        assert torch.equal(cuda_ext.w4_linear(x, w4), want)
        assert L.device_status(0) == 0


@pytest.mark.parametrize("m", [3, 40, 200])
def test_chain_with_missing_codes_times_out(cuda_dev, m):
    layers = [make(k, n, torch.bfloat16, 128, False) for k, n in ((256, 512), (512, 136), (136, 64))]
    ws = [cuda_ext.w4_pack(*layer, group=128) for layer in layers]
    x, kw = rows(m, 256, torch.bfloat16), dict(acts=[L.ACT_RELU, L.ACT_RELU, L.ACT_NONE])
    want = cuda_ext.w4_mlp(x, ws, [None] * 3, **kw)
    assert L.device_status(0, clear=True) == 0
    try:
        L.set_timeout_ns(5_000_000)
        L.set_fault_injection(1)
        cuda_ext.w4_mlp(x, ws, [None] * 3, **kw)
        torch.cuda.synchronize()
    finally:
        L.set_fault_injection(0)
        L.set_timeout_ns(0)
    assert L.device_status(0, clear=True) in (0x100, 0x200, 0x300)
    assert torch.equal(cuda_ext.w4_mlp(x, ws, [None] * 3, **kw), want)
    assert L.device_status(0) == 0
