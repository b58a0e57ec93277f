"""Block-128 fp8: quantisation, block-scaled products, the fp8 linear and AdamW over lists.

Every operator is compared with a plain implementation in 64 bits written here; the CPU
parametrisations run the PyTorch reference, the ``gpu`` ones the sm_100a kernels.

Tolerances.  Codes, scales and 8-bit moments are defined bit for bit and compared exactly.  A
product of quantised operands differs from its 64-bit value by the rounding of its output
(2^-9 relative for bf16, 2^-24 for fp32) and by the fp32 accumulation: K / 32 steps of 32
products, each taken to at least 22 bits below the largest partial sum, so by at most
(K / 32 + 32) 2^-22 times the sum of the products' magnitudes.
"""
import math

import pytest
import torch

from osp_next_b200 import ops
from osp_next_b200.parallel.optim import FusedAdamW
from osp_next_b200.quant import FP8Linear, fp8_linear, freeze_fp8_weights

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
GPU = [pytest.param("cuda", marks=pytest.mark.gpu)]


def _randn(*shape, device, seed=0, dtype=torch.float32, spread=0.7):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(shape[-1], generator=g))
    return x.to(device=device, dtype=dtype)


# ----------------------------------------------------------------------------- 64-bit forms

def _two_to(k):
    return ((k.long() + 1023) << 52).view(torch.float64)


def quantize64(x, block_rows=1):
    """(e4m3 values, scale exponents per block) of a matrix, in 64 bits."""
    x = x.detach().double().cpu()
    R, K = x.shape
    rt, kb = -(-R // block_rows), -(-K // 128)
    full = torch.zeros(rt * block_rows, kb * 128, dtype=torch.float64)
    full[:R, :K] = x
    t = full.view(rt, block_rows, kb, 128)
    top = torch.where(torch.isfinite(t), t.abs(), torch.zeros_like(t)).amax((1, 3), keepdim=True)
    k = torch.full_like(top, -126)
    for e in range(-126, 120):                       # the definition: raise until it fits
        k = torch.where(top > 448 * 2.0 ** e, torch.full_like(k, e + 1), k)
    y = t / _two_to(k)
    _, e = torch.frexp(y.abs().clamp(min=2.0 ** -6))
    step = _two_to(e - 4)
    q = torch.where(torch.isfinite(y), torch.round(y / step) * step, torch.full_like(y, math.nan))
    k = k.expand(rt, block_rows, kb, 1).reshape(-1, kb)[:R]
    return q.reshape(rt * block_rows, -1)[:R], k


def check_quantized(t, x, block_rows):
    R, K = x.shape
    q, k = quantize64(x, block_rows)
    assert tuple(t.shape) == (R, K) and t.data.dtype == torch.float8_e4m3fn
    assert tuple(t.data.shape) == (R, -(-K // 128) * 128)
    got = t.data.cpu().double()
    assert torch.equal(got.isnan(), q.isnan())
    assert torch.equal(got.nan_to_num(9e9), q.nan_to_num(9e9))
    want = torch.zeros(t.scale.shape, dtype=torch.uint8)
    r, b = torch.meshgrid(torch.arange(R), torch.arange(q.shape[1] // 128), indexing="ij")
    want[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = (k + 127).to(torch.uint8)
    assert torch.equal(t.scale.cpu(), want)


# ----------------------------------------------------------------------------- quantisation

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,K", [(1, 1), (1, 128), (3, 129), (128, 512), (130, 777), (257, 1040), (1, 5120)])
def test_quantize(device, dtype, R, K):
    x = _randn(R, K, device=device, seed=R + K, dtype=dtype)
    check_quantized(ops.fp8_quantize(x), x, 1)
    check_quantized(ops.fp8_quantize(x, layout="cols"), x.t(), 1)
    for block in (1, 128):
        rows, cols = ops.fp8_quantize(x, block_rows=block, layout="both")
        check_quantized(rows, x, block)
        check_quantized(cols, x.t(), block)
    check_quantized(ops.fp8_quantize(x, block_rows=128), x, 128)
    check_quantized(ops.fp8_quantize(x, block_rows=128, layout="cols"), x.t(), 128)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_strides(device, dtype):
    buf = _randn(140, 901, device=device, dtype=dtype)
    views = [buf[:, :300], buf[:, 8:308], buf[:, 3:700], buf[5:, 64:192], buf.t(), buf.t()[3:200, 1:], buf[::2, :256],
             buf[:, ::3], buf[:1].expand(70, 901), buf[:, :1].expand(140, 300)]
    for x in views:
        for layout in ("rows", "cols"):
            t = ops.fp8_quantize(x, layout=layout)
            check_quantized(t, x if layout == "rows" else x.t(), 1)
        check_quantized(ops.fp8_quantize(x, block_rows=128), x, 128)


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_extremes(device):
    """Zeros, the range's ends, exact block maxima, halves between codes, and non-finite values."""
    big = torch.finfo(torch.float32).max
    rows = [torch.zeros(300), torch.full((300,), 448.0), torch.full((300,), 448.0001), torch.full((300,), big),
            torch.full((300,), 1e-45), torch.full((300,), -2.0 ** -126), torch.linspace(-448, 448, 300),
            torch.arange(300) / 512.0, 2.0 ** torch.linspace(-40, 30, 300), torch.full((300,), math.nan),
            torch.full((300,), -math.inf)]
    mixed = _randn(4, 300, device="cpu", seed=3)
    mixed[0, 5], mixed[1, 128], mixed[2, 299], mixed[3, :128] = math.inf, math.nan, -math.inf, math.nan
    x = torch.cat([torch.stack(rows), mixed]).to(device)
    for block in (1, 128):
        rows_, cols = ops.fp8_quantize(x, block_rows=block, layout="both")
        check_quantized(rows_, x, block)
        check_quantized(cols, x.t(), block)
    check_quantized(ops.fp8_quantize(x), x, 1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,K", [(1, 1), (5, 130), (128, 256), (300, 515), (1000, 72)])
def test_quantize_with_sums(device, dtype, R, K):
    x = _randn(R, K + 8, device=device, seed=R, dtype=dtype)
    for v in (x[:, :K], x[:, 8:], x.t()[:K].t()):
        rows, cols, sums = ops.fp8_quantize_with_sums(v)
        check_quantized(rows, v, 1)
        check_quantized(cols, v.t(), 1)
        # R additions in fp32
        assert bool(((sums.double() - v.double().sum(0)).abs() <= R * 2.0 ** -24 * v.double().abs().sum(0)).all())
    x[R // 2, 0], x[0, K // 2] = math.inf, math.nan
    bad = ops.fp8_quantize_with_sums(x[:, :K])[2]
    assert torch.equal(bad, x[:, :K].float().sum(0)) or torch.equal(bad.isfinite(), x[:, :K].float().sum(0).isfinite())


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_empty(device):
    for R, K in ((0, 5), (5, 0), (0, 0)):
        t = ops.fp8_quantize(torch.zeros(R, K, device=device))
        assert tuple(t.shape) == (R, K) and t.data.numel() == 0


@pytest.mark.parametrize("device", DEVICES)
def test_dequantize(device):
    x = _randn(130, 300, device=device)
    q, k = quantize64(x)
    want = (q * _two_to(k).repeat_interleave(128, 1))[:, :300]
    assert torch.equal(ops.fp8_quantize(x).dequantize().cpu().double(), want)


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_refusals(device):
    x = torch.zeros(4, 4, device=device)
    with pytest.raises(ValueError):
        ops.fp8_quantize(x[0])
    with pytest.raises(TypeError):
        ops.fp8_quantize(x.double())
    with pytest.raises(ValueError):
        ops.fp8_quantize(x, block_rows=64)
    with pytest.raises(ValueError):
        ops.fp8_quantize(x, layout="row")


# ----------------------------------------------------------------------------- products

def _gelu64(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def check_product(y, a, b, bias=None, act=None):
    """y against the 64-bit product of the quantised operands."""
    A, B = a.dequantize().double().cpu(), b.dequantize().double().cpu()
    want, mag = A @ B.t(), A.abs() @ B.abs().t()
    if bias is not None:
        want, mag = want + bias.double().cpu(), mag + bias.double().cpu().abs()
    err = (a.cols / 32 + 32) * 2.0 ** -22 * mag
    if act:                                           # slope of GELU below 1.13; its own fp32 rounding
        want, err = _gelu64(want), 1.13 * err + 2.0 ** -21 * (1 + want.abs())
    err = err + (2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -23) * want.abs() + 1e-38
    got = y.double().cpu()
    assert got.shape == want.shape
    assert bool(((got - want).abs() <= err).all()), float(((got - want).abs() / err).max())


PRODUCTS = [(1, 16, 64), (1, 300, 5120), (2, 129, 640), (7, 1000, 130), (33, 128, 2048), (64, 512, 128),
            (65, 640, 384), (128, 256, 512), (130, 64, 900), (200, 72, 1111), (300, 777, 1024), (513, 1536, 640),
            (1025, 250, 257), (2500, 2304, 512), (4700, 1300, 1111), (19000, 200, 129), (12, 1, 128), (5, 13824, 200)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_matmul(device, M, N, K):
    x = _randn(M, K, device=device, seed=M, dtype=torch.bfloat16)
    w = _randn(N, K, device=device, seed=N, spread=0.2) / math.sqrt(K)
    bias = _randn(N, device=device, seed=K)
    wq, xq = ops.fp8_quantize(w, block_rows=128), ops.fp8_quantize(x)
    for out_dtype in (torch.bfloat16, torch.float32):
        y = ops.fp8_matmul(x, wq, out_dtype=out_dtype)
        assert y.dtype == out_dtype
        check_product(y, xq, wq)
        check_product(ops.fp8_matmul(xq, wq, bias, "gelu_tanh", out_dtype), xq, wq, bias, "gelu_tanh")
    y, pre = ops.fp8_matmul(x, wq, bias, "gelu_tanh", aux=True)
    check_product(pre, xq, wq, bias)
    check_product(y, xq, wq, bias, "gelu_tanh")


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(3, 130, 20160), (64, 256, 9000), (40, 5120, 5120), (256, 300, 14040),
                                   (700, 512, 20161), (1000, 64, 5120), (3000, 2304, 2200)])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_matmul_long_sums_in_fp32(M, N, K, act):
    """Sums of one sign, where cutting each of the K / 32 steps would add up: runs of 64 steps cut
    the growing sum by at most 2^-23 of it each, half of that in the mean and half a run's sum
    on average, 64 / 4 * 2^-23 = 2^-19 in all; as much again for the additions of the runs."""
    x = _randn(M, K, device="cuda", seed=M, dtype=torch.bfloat16).abs()
    w = _randn(N, K, device="cuda", seed=N, spread=0.2).abs() / K
    bias = _randn(N, device="cuda").abs()
    wq, xq = ops.fp8_quantize(w, block_rows=128), ops.fp8_quantize(x)
    want = xq.dequantize().double() @ wq.dequantize().double().t() + bias.double()
    y, pre = ops.fp8_matmul(x, wq, bias, act, torch.float32, aux=True)
    if act:
        want_pre, want = want, _gelu64(want)
        assert bool(((pre.double() - want_pre).abs() <= 2.0 ** -8 * want_pre).all())
    assert ((y.double() - want).norm() / want.norm()).item() < 2.0 ** -18
    again = ops.fp8_matmul(x, wq, bias, act, torch.float32)
    assert torch.equal(again, y)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,N,K", [(1, 200, 700), (70, 130, 515), (300, 260, 300)])
def test_matmul_scales_by_row_and_block(device, M, N, K):
    """Row scales of both operands that differ by 2^40 from block to block."""
    g = torch.Generator().manual_seed(5)
    kb = -(-K // 128)

    def wild(R):
        e = torch.randint(-20, 21, (R, kb), generator=g).repeat_interleave(128, 1)[:, :K]
        return (torch.randn(R, K, generator=g) * 2.0 ** e).to(device)
    a, b = ops.fp8_quantize(wild(M)), ops.fp8_quantize(wild(N))
    check_product(ops.fp8_matmul(a, b, out_dtype=torch.float32), a, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M", [1, 3, 40, 100, 300])
def test_matmul_nan_stays_in_its_row(device, M):
    x = _randn(M, 384, device=device, dtype=torch.bfloat16)
    w = _randn(96, 384, device=device, seed=1)
    x[M // 2, 200], w[17, 3] = math.inf, math.nan
    y = ops.fp8_matmul(x, ops.fp8_quantize(w), out_dtype=torch.float32)
    bad = torch.zeros(M, 96, dtype=torch.bool)
    bad[M // 2], bad[:, 17] = True, True
    assert torch.equal(y.isnan().cpu(), bad) and bool(y[~bad.to(y.device)].isfinite().all())


@pytest.mark.parametrize("device", DEVICES)
def test_matmul_batches_and_empty(device):
    w = ops.fp8_quantize(_randn(24, 130, device=device), block_rows=128)
    x = _randn(2, 3, 130, device=device, dtype=torch.bfloat16)
    y = ops.fp8_matmul(x, w)
    assert y.shape == (2, 3, 24) and torch.equal(y, ops.fp8_matmul(x.view(6, 130), w).view(2, 3, 24))
    assert ops.fp8_matmul(x[0, 0], w).shape == (24,)
    assert ops.fp8_matmul(x[:, :0], w).shape == (2, 0, 24)
    b = torch.arange(4.0, device=device)
    none = ops.fp8_matmul(torch.zeros(3, 0, device=device), ops.fp8_quantize(torch.zeros(4, 0, device=device)), b)
    assert torch.equal(none.float(), b.expand(3, 4))
    # strided and sliced activations
    buf = _randn(50, 400, device=device, dtype=torch.bfloat16)
    v = buf[:, 7:137]
    assert torch.equal(ops.fp8_matmul(v, w), ops.fp8_matmul(v.contiguous(), w))


@pytest.mark.parametrize("device", DEVICES)
def test_matmul_refusals(device):
    w = ops.fp8_quantize(torch.zeros(8, 64, device=device), block_rows=128)
    x = torch.zeros(2, 64, device=device)
    with pytest.raises(TypeError):
        ops.fp8_matmul(x, x)
    with pytest.raises(ValueError):
        ops.fp8_matmul(x[:, :32], w)
    with pytest.raises(ValueError):
        ops.fp8_matmul(ops.fp8_quantize(x[:, :32]), w)
    with pytest.raises(ValueError):
        ops.fp8_matmul(x, w, bias=torch.zeros(7, device=device))
    with pytest.raises(ValueError):
        ops.fp8_matmul(x, w, act="relu")
    with pytest.raises(TypeError):
        ops.fp8_matmul(x, w, out_dtype=torch.float16)


@pytest.mark.gpu
def test_matmul_kernel_refuses_wrong_buffers():
    w = ops.fp8_quantize(torch.zeros(8, 64, device="cuda"), block_rows=128)
    x = ops.fp8_quantize(torch.zeros(200, 64, device="cuda"))
    for bad in (ops.Fp8Tensor(x.data, x.scale[:1], 200, 64), ops.Fp8Tensor(x.data[:, :64], x.scale, 200, 64),
                ops.Fp8Tensor(x.data.view(torch.uint8), x.scale, 200, 64), ops.Fp8Tensor(x.data, x.scale.cpu(), 200, 64)):
        with pytest.raises(RuntimeError):
            ops.fp8_matmul(bad, w)


@pytest.mark.gpu
def test_matmul_on_another_stream_and_in_a_graph():
    x = _randn(300, 512, device="cuda", dtype=torch.bfloat16)
    w = ops.fp8_quantize(_randn(512, 512, device="cuda", seed=1), block_rows=128)
    want = [ops.fp8_matmul(x, w), ops.fp8_matmul(x[:2], w)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ops.fp8_matmul(x, w), ops.fp8_matmul(x[:2], w)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    xs = torch.zeros_like(x)
    with torch.cuda.graph(graph):
        ys = [ops.fp8_matmul(xs, w), ops.fp8_matmul(xs[:2], w)]
    xs.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ys, want))
    ops.check_device_errors()


@pytest.mark.gpu
def test_matmul_repeats_bit_for_bit():
    for M in (1, 5, 60, 500):
        x = _randn(M, 1536, device="cuda", dtype=torch.bfloat16)
        w = ops.fp8_quantize(_randn(1500, 1536, device="cuda", seed=1), block_rows=128)
        y = ops.fp8_matmul(x, w, out_dtype=torch.float32)
        assert all(torch.equal(y, ops.fp8_matmul(x, w, out_dtype=torch.float32)) for _ in range(20))


# ----------------------------------------------------------------------------- fp8 linear, autograd

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,N,K", [(1, 40, 130), (70, 96, 256), (300, 260, 129), (515, 384, 640)])
@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("with_bias", [True, False])
def test_linear_gradients(device, M, N, K, wdtype, with_bias):
    """y, dx, dW, db against the formulas on the quantised operands."""
    x = _randn(M, K, device=device, seed=M, dtype=torch.bfloat16).requires_grad_()
    w = (_randn(N, K, device=device, seed=N, spread=0.2) / math.sqrt(K)).to(wdtype).requires_grad_()
    bias = _randn(N, device=device, seed=1).requires_grad_() if with_bias else None
    dy = _randn(M, N, device=device, seed=2, dtype=torch.bfloat16)
    y = fp8_linear(x, w, bias)
    grads = torch.autograd.grad(y, [x, w] + ([bias] if with_bias else []), dy)
    wr, wc = ops.fp8_quantize(w, block_rows=128, layout="both")
    xr, xc = ops.fp8_quantize(x, layout="both")
    gr, gc = ops.fp8_quantize(dy, layout="both")
    check_product(y.detach(), xr, wr, bias.detach() if with_bias else None)
    check_product(grads[0], gr, wc)
    check_product(grads[1], gc, xc)
    assert grads[0].dtype == x.dtype and grads[1].dtype == wdtype
    if with_bias:
        want = dy.double().sum(0)
        assert bool(((grads[2].double() - want).abs() <= M * 2.0 ** -24 * dy.double().abs().sum(0)).all())


@pytest.mark.parametrize("device", DEVICES)
def test_linear_gradient_against_differences(device):
    """On grid values (small integers: quantisation changes nothing, sums are exact) the map is
    linear, so central differences of <y, dy> with steps of 1 are its derivative exactly."""
    g = torch.Generator().manual_seed(0)
    M, N, K = 3, 5, 140

    def grid(*s):
        t = torch.randint(-4, 5, s, generator=g).float()
        return t.to(device)
    x, w, b, dy = grid(M, K), grid(N, K), grid(N), grid(M, N)
    args = [t.clone().requires_grad_() for t in (x, w, b)]
    y = fp8_linear(*args)
    grads = torch.autograd.grad(y, args, dy.to(y.dtype))

    def f(*t):
        wq = ops.fp8_quantize(t[1], block_rows=128)
        return (ops.fp8_matmul(t[0], wq, t[2], out_dtype=torch.float32).double() * dy.double()).sum().item()
    for n, t in enumerate((x, w, b)):
        for i in range(0, t.numel(), 37):
            lo, hi = t.clone(), t.clone()
            lo.view(-1)[i] -= 1
            hi.view(-1)[i] += 1
            parts = [x, w, b]
            d = (f(*parts[:n], hi, *parts[n + 1:]) - f(*parts[:n], lo, *parts[n + 1:])) / 2
            assert d == grads[n].view(-1)[i].item()


@pytest.mark.parametrize("device", DEVICES)
def test_linear_gelu(device):
    x = _randn(70, 256, device=device, dtype=torch.bfloat16).requires_grad_()
    w = (_randn(96, 256, device=device, seed=1) / 16).requires_grad_()
    b = _randn(96, device=device, seed=2).requires_grad_()
    y = fp8_linear(x, w, b, act="gelu_tanh")
    wr, wc = ops.fp8_quantize(w, block_rows=128, layout="both")
    check_product(y.detach(), ops.fp8_quantize(x), wr, b.detach(), "gelu_tanh")
    dy = _randn(70, 96, device=device, seed=3, dtype=torch.bfloat16)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    # through the bf16 pre-activation: d = dy gelu'(pre), rounded to bf16 (2^-9, and as much again
    # through a code that the rounding moved: one e4m3 step, 2^-3, of few elements)
    pre = ops.fp8_matmul(x.detach(), wr, b.detach(), out_dtype=torch.float32).bfloat16().double()
    pre.requires_grad_()
    (d,) = torch.autograd.grad(_gelu64(pre), pre, dy.double())
    want = ops.fp8_quantize(d.bfloat16()).dequantize().double() @ wc.dequantize().double().t()
    assert ((dx.double() - want).norm() / want.norm()).item() < 2.0 ** -7
    assert dw.shape == w.shape and bool(dw.isfinite().all())


@pytest.mark.parametrize("device", DEVICES)
def test_linear_partial_gradients_and_shapes(device):
    w = _randn(40, 130, device=device)
    for needs in ((True, False, False), (False, True, False), (False, False, True)):
        x = _randn(2, 3, 130, device=device, dtype=torch.bfloat16).requires_grad_(needs[0])
        ww = w.clone().requires_grad_(needs[1])
        b = torch.zeros(40, device=device, requires_grad=needs[2])
        y = fp8_linear(x, ww, b)
        assert y.shape == (2, 3, 40)
        y.float().square().sum().backward()
        for t, n in zip((x, ww, b), needs):
            assert (t.grad is not None) == n and (not n or (t.grad.shape == t.shape and t.grad.dtype == t.dtype))
    with pytest.raises(ValueError):
        fp8_linear(x[..., :100], w)
    with pytest.raises(ValueError):
        fp8_linear(x, w, torch.zeros(39, device=device))
    # no tokens: an empty output and a zero weight gradient
    x = torch.zeros(0, 130, device=device, dtype=torch.bfloat16)
    ww = w.clone().requires_grad_()
    fp8_linear(x, ww).float().sum().backward()
    assert torch.equal(ww.grad, torch.zeros_like(ww))


@pytest.mark.parametrize("device", DEVICES)
def test_linear_module_freezing(device):
    torch.manual_seed(0)
    layer = FP8Linear(64, 32, device=device)
    x = _randn(5, 64, device=device, dtype=torch.bfloat16)
    with torch.no_grad():
        y0 = layer(x)
        freeze_fp8_weights(layer)
        assert torch.equal(layer(x), y0)
        layer.weight.data.mul_(3)                    # frozen: the quantised copy is what is used
        assert torch.equal(layer(x), y0)
        layer.thaw_weight()
        y1 = layer(x)
        assert not torch.equal(y1, y0)
        layer.freeze_weight()
        layer.load_state_dict({k: v * 2 for k, v in layer.state_dict().items()})
        assert not torch.equal(layer(x), y1)
        layer.freeze_weight()
        layer.train()
        assert layer._frozen is None
    assert layer(x).requires_grad


# ----------------------------------------------------------------------------- AdamW on lists

HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1)
SIZES = [1, 5, 127, 128, 129, 1000, 4096, 4097, 70001]


def _lists(sizes, device, pdtype, gdtype, seed=0):
    p = [_randn(n, device=device, seed=seed + i, dtype=pdtype, spread=0) for i, n in enumerate(sizes)]
    g = [_randn(n, device=device, seed=seed + 50 + i, dtype=gdtype, spread=1.5) * 1e-3 for i, n in enumerate(sizes)]
    return p, [t.to(gdtype) for t in g]


def _adamw64(p, g, m, v, step, grad_scale, lr, beta1, beta2, eps, weight_decay):
    g = g.double() * grad_scale
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    upd = m / (1 - beta1 ** step) / (v.div(1 - beta2 ** step).sqrt() + eps)
    return p.double() * (1 - lr * weight_decay) - lr * upd, m, v


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("pdtype,gdtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                           (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_adamw32(device, pdtype, gdtype):
    p, g = _lists(SIZES, device, pdtype, gdtype)
    m, v = [torch.zeros(n, device=device) for n in SIZES], [torch.zeros(n, device=device) for n in SIZES]
    for step in (1, 2, 3):
        want = [_adamw64(a, b, c.double(), d.double(), step, 0.5, **HYPER) for a, b, c, d in zip(p, g, m, v)]
        ops.adamw_multi_(p, g, m, v, step=step, grad_scale=0.5, **HYPER)
        for a, c, d, (wp, wm, wv) in zip(p, m, v, want):
            # a few fp32 roundings per value; 1 - b^t is formed in fp32 (2^-24 of 1 over 1e-3)
            rp = 2.0 ** -8 if pdtype == torch.bfloat16 else 2.0 ** -22
            assert bool(((a.double() - wp).abs() <= rp * wp.abs() + 1e-2 * 2.0 ** -13).all())
            assert bool(((c.double() - wm).abs() <= 2.0 ** -21 * (wm.abs() + 1e-3)).all())
            assert bool(((d.double() - wv).abs() <= 2.0 ** -21 * wv.abs() + 1e-30).all())


@pytest.mark.gpu
@pytest.mark.parametrize("gdtype", [torch.float32, torch.bfloat16])
def test_adamw32_agrees_with_the_per_tensor_kernel(gdtype):
    """Up to that kernel's 1 - b, formed from the fp32 b: off by 2^-24 over 0.001, 2^-14."""
    p, g = _lists(SIZES, "cuda", torch.float32, gdtype)
    m, v = [torch.zeros_like(t) for t in p], [torch.zeros_like(t) for t in p]
    p1, m1, v1 = ([t.clone() for t in x] for x in (p, m, v))
    for step in (1, 2, 7):
        ops.adamw_multi_(p, g, m, v, step=step, grad_scale=0.3, **HYPER)
        for a, b, c, d in zip(p1, g, m1, v1):
            ops.adamw_(a, b, c, d, HYPER["lr"], 0.9, 0.999, HYPER["eps"], HYPER["weight_decay"], step, 0.3)
    for x, y, slack in ((p, p1, 3e-2 * 2.0 ** -13), (m, m1, 1e-8), (v, v1, 0.0)):
        for a, b in zip(x, y):
            assert bool(((a - b).abs() <= 2.0 ** -13 * b.abs() + slack).all())


def _neighbours(x, mant, low, top):
    """The format's values below and above |x| (3 mantissa bits, least normal ``low``), in 64 bits."""
    a = x.abs()
    _, e = torch.frexp(a.clamp(min=low))
    step = _two_to(e - 1 - mant)
    lo = torch.floor(a / step) * step
    return lo, torch.where(lo == a, lo, lo + step)


def _check_state8(m8, v8, ms, vs, m, v):
    """8-bit moments are one of the two neighbours of the exact fp32 moments m, v."""
    n = m.numel()
    nb = -(-n // 128)

    def blocks(t):
        out = torch.zeros(nb * 128, dtype=torch.float64)
        out[:n] = t.double().cpu()
        return out.view(nb, 128)
    got_m, got_v = (t.double().cpu() for t in ops.adamw8_decode(m8, v8, ms, vs))
    for x, got, s, top, low, keep in ((m, got_m, ms, 448.0, 2.0 ** -6, False), (v, got_v, vs, 61440.0, 2.0 ** -14, True)):
        b = blocks(x)
        k = torch.full((nb,), -126)
        for e in range(-126, 60):
            k = torch.where(b.abs().amax(1) > top * 2.0 ** e, torch.full_like(k, e + 1), k)
        assert torch.equal(s.cpu().long(), k.long() + 127)
        sc = _two_to(k)[:, None].expand(nb, 128).reshape(-1)[:n]
        y = x.double().cpu() / sc
        lo, hi = _neighbours(y, 3, low, top)
        q = got / sc
        ok = (q.abs() == lo) | (q.abs() == hi)
        if keep:                                      # a positive v is never stored as zero
            ok &= (q > 0) == (y > 0)
        assert bool(ok.all()) and bool(((q == 0) | (torch.sign(q) == torch.sign(y))).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gdtype", [torch.float32, torch.bfloat16])
def test_adamw8(device, gdtype):
    p, g = _lists(SIZES, device, torch.float32, gdtype)
    g[5][128:256] = 0                                 # a block without gradients
    state = [ops.adamw8_state(t) for t in p]
    m, v, ms, vs = (list(x) for x in zip(*state))
    b1, b2 = (torch.tensor(x, dtype=torch.float32).item() for x in (0.9, 0.999))
    c1, c2 = (torch.tensor(x, dtype=torch.float32).item() for x in (1 - 0.9, 1 - 0.999))
    for step in (1, 2, 3):
        old = [tuple(t.double().cpu() for t in ops.adamw8_decode(*x)) for x in zip(m, v, ms, vs)]
        want = [_adamw64(a.cpu(), b.cpu(), c, d, step, 0.5, **HYPER) for a, b, (c, d) in zip(p, g, old)]
        ops.adamw_multi_(p, g, m, v, ms, vs, step=step, grad_scale=0.5, seed=step, **HYPER)
        for i, (wp, wm, wv) in enumerate(want):
            assert bool(((p[i].double().cpu() - wp).abs() <= 2.0 ** -22 * wp.abs() + 1e-2 * 2.0 ** -13).all())
            # the fp32 moments before rounding, with the formula's own roundings
            g32 = (g[i].float() * 0.5).cpu()
            m32 = old[i][0].float() * b1 + g32 * c1
            v32 = old[i][1].float() * b2 + (g32 * g32) * c2
            _check_state8(m[i], v[i], ms[i], vs[i], m32, v32)


@pytest.mark.gpu
def test_adamw8_kernel_equals_the_reference():
    """Same seed, same bits: codes and scales of the kernel and of the CPU form agree."""
    p, g = _lists(SIZES, "cpu", torch.float32, torch.float32)
    host = [p, g] + [list(x) for x in zip(*(ops.adamw8_state(t) for t in p))]
    dev = [[t.cuda() for t in x] for x in host]
    for step in (1, 2, 3):
        for lists in (host, dev):
            ops.adamw_multi_(*lists, step=step, grad_scale=0.7, seed=41 * step, **HYPER)
        for a, b in zip(host[2:], dev[2:]):
            assert all(torch.equal(x.view(torch.uint8), y.cpu().view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("device", DEVICES)
def test_adamw8_rounding_is_unbiased(device):
    """The mean over seeds of a stored moment approaches the moment: 400 draws of a value whose
    rounding moves it by at most one step s have a standard deviation below s / 2 / 20."""
    n = 128
    p, g = [torch.zeros(n, device=device)], [torch.linspace(0.1, 1, n, device=device)]
    sums = [torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)]
    for seed in range(400):
        m, v, ms, vs = ([t] for t in ops.adamw8_state(p[0]))
        ops.adamw_multi_(p, g, m, v, ms, vs, step=1, seed=seed, **HYPER)
        for acc, t in zip(sums, ops.adamw8_decode(m[0], v[0], ms[0], vs[0])):
            acc += t.double().cpu() / 400
    gd = g[0].double().cpu()
    for got, want in ((sums[0], 0.1 * gd), (sums[1], 0.001 * gd * gd)):
        step = want / 8
        assert bool(((got - want).abs() < 5 * step / 40).all())


@pytest.mark.parametrize("device", DEVICES)
def test_adamw8_small_second_moment_decays(device):
    """With zero gradients v falls by beta2 each step on average: nearest rounding would hold it."""
    n = 128 * 64
    p, g = [torch.zeros(n, device=device)], [torch.ones(n, device=device)]
    m, v, ms, vs = ([t] for t in ops.adamw8_state(p[0]))
    ops.adamw_multi_(p, g, m, v, ms, vs, step=1, seed=0, **HYPER)
    v0 = ops.adamw8_decode(m[0], v[0], ms[0], vs[0])[1].double().mean().item()
    g[0].zero_()
    for step in range(2, 102):
        ops.adamw_multi_(p, g, m, v, ms, vs, step=step, seed=step, **HYPER)
    v1 = ops.adamw8_decode(m[0], v[0], ms[0], vs[0])[1].double().mean().item()
    # a walk of 100 steps of at most 1/8 with p(1 - p) <= 0.02, over 8192 elements
    assert abs(v1 / v0 - 0.999 ** 100) < 5 * 0.125 * math.sqrt(100 * 0.02 / n) * 1.2


@pytest.mark.parametrize("device", DEVICES)
def test_adamw8_non_finite(device):
    """A NaN or infinite gradient spoils its own element, as with fp32 moments, and no other."""
    p, g = [torch.ones(300, device=device)], [torch.ones(300, device=device)]
    g[0][7], g[0][200] = math.nan, math.inf
    m, v, ms, vs = ([t] for t in ops.adamw8_state(p[0]))
    ops.adamw_multi_(p, g, m, v, ms, vs, step=1, seed=3, **HYPER)
    md, vd = ops.adamw8_decode(m[0], v[0], ms[0], vs[0])
    bad = torch.zeros(300, dtype=torch.bool)
    bad[7] = bad[200] = True
    for t in (md, vd):
        assert torch.equal(t.isfinite().cpu(), ~bad)
    assert torch.equal(p[0].isnan().cpu(), bad)


@pytest.mark.gpu
def test_adamw_misaligned_and_many():
    """Tensors that start anywhere, zero-length ones, and more than fit one launch."""
    sizes = [1 + 37 * i % 400 for i in range(1100)] + [0, 9]
    total = sum(sizes) + len(sizes)
    flat = [_randn(total, device="cuda", seed=i, spread=0) for i in range(2)]
    offs = [0]
    for n in sizes:
        offs.append(offs[-1] + n + 1)
    p, g = ([f[o:o + n] for o, n in zip(offs, sizes)] for f in flat)
    host = [[t.cpu().clone() for t in x] for x in (p, g)]
    bufs = [torch.zeros(total, dtype=torch.uint8, device="cuda") for _ in range(2)]
    state = [ops.adamw8_state(t) for t in p]
    m = [bufs[0][o:o + n].view(torch.float8_e4m3fn) for o, n in zip(offs, sizes)]
    v = [bufs[1][o:o + n] for o, n in zip(offs, sizes)]
    ms, vs = [s[2] for s in state], [s[3] for s in state]
    dev = [p, g, m, v, ms, vs]
    host += [[t.cpu().clone() for t in x] for x in dev[2:]]
    for step in (1, 2):
        for lists in (dev, host):
            ops.adamw_multi_(*lists, step=step, seed=9, **HYPER)
    for a, b in zip(dev[2:], host[2:]):
        assert all(torch.equal(x.cpu().view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))
    for a, b in zip(p, host[0]):
        assert bool(((a.cpu() - b).abs() <= 2.0 ** -21 * (b.abs() + 1)).all())


@pytest.mark.parametrize("device", DEVICES)
def test_adamw_refusals(device):
    z = lambda n=4: [torch.zeros(n, device=device)]  # noqa: E731
    with pytest.raises(ValueError):
        ops.adamw_multi_(z(), z() + z(), z(), z(), step=1, **HYPER)
    with pytest.raises(ValueError):
        ops.adamw_multi_(z(), z(), z(), z(), step=0, **HYPER)
    with pytest.raises(ValueError):
        ops.adamw_multi_(z(), z(), z(), z(), exp_avg_scales=z(), step=1, **HYPER)
    ops.adamw_multi_([], [], [], [], step=1, **HYPER)
    if device == "cuda":
        for bad in ([z(), z(5), z(), z()], [z(), z(), z(), [torch.zeros(4, device=device).half()]],
                    [[torch.zeros(4, 4, device=device).t()[:2]], z(8), z(8), z(8)],
                    [z(), [torch.zeros(4)], z(), z()]):
            with pytest.raises(RuntimeError):
                ops.adamw_multi_(*bad, step=1, **HYPER)
