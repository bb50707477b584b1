"""8-bit block quantisation, its product and the linear layer on the GPU, against plain formulas in 64 bits.

Codes and scales are defined exactly (power-of-two scales, one rounding), so they must be equal.  Products: an MMA adds
32 exact products to the fp32 accumulator and keeps at least 22 bits below its largest addend, so after K / 32 of them an
element is off by at most (K / 32 + 1) 2^-22 of the sum of its products' magnitudes; results in bf16 add half a step, 2^-8
of the value.
"""

import pytest
import torch

from mvp_engine import ops
from mvp_engine.ops import _ext
from mvp_engine.ops.fp8 import _quantize_plain

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def rand(shape, seed=0, dtype=torch.bfloat16, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[0], 1, generator=g))
    return x.to(dtype).cuda()


def same(a, b):
    """Equal matrices: bytes of codes (NaNs by position) and of scales."""
    assert a.shape == b.shape and a.dtype == b.dtype and a.data.shape == b.data.shape
    x, y = a.data.cpu().float(), b.data.cpu().float()
    assert torch.equal(torch.isnan(x), torch.isnan(y))
    assert torch.equal(torch.nan_to_num(x), torch.nan_to_num(y))
    assert torch.equal(a.scale.cpu(), b.scale.cpu())


SHAPES = [(1, 1), (1, 128), (128, 1), (7, 8), (8, 130), (127, 129), (129, 127), (128, 512), (300, 520), (257, 1000),
          (640, 513)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("src,dtype", [(torch.bfloat16, E4M3), (torch.float32, E4M3), (torch.bfloat16, E5M2)])
def test_quantize(shape, block, src, dtype):
    x = rand(shape, shape[0] + 31 * shape[1], src)
    q, t = ops.quantize_fp8(x, block, rows=True, columns=True, dtype=dtype)
    same(q, _quantize_plain(x.cpu(), block == "tile", dtype))
    same(t, _quantize_plain(x.cpu().t(), block == "tile", dtype))
    only_q, none = ops.quantize_fp8(x, block, dtype=dtype)
    none2, only_t = ops.quantize_fp8(x, block, rows=False, columns=True, dtype=dtype)
    assert none is None and none2 is None
    same(only_q, q)
    same(only_t, t)


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
def test_quantize_extremes(src):
    """Zero blocks, the smallest and largest values, borders of the range, values that are not finite."""
    x = torch.zeros(300, 400)
    x[1] = 448.0
    x[2] = 448.0 * 2.0**-20
    x[3] = 452.0
    x[4] = torch.finfo(src).max
    x[5] = torch.finfo(src).tiny
    x[6] = torch.finfo(src).smallest_normal / 128
    x[7, 3] = float("nan")
    x[8, 200] = float("inf")
    x[9, 399] = -float("inf")
    x[10:200] = rand((190, 400), 1).float().cpu()
    x[250, 7] = 1e-30
    x = x.to(src)
    for block in ("row", "tile"):
        q, t = ops.quantize_fp8(x.cuda(), block, rows=True, columns=True)
        same(q, _quantize_plain(x, block == "tile", E4M3))
        same(t, _quantize_plain(x.t(), block == "tile", E4M3))


def test_quantize_strides():
    base = rand((300, 700), 3)
    for x in (base[:, 1:301], base[::2, 5:600], base[:, :1], base.t(), base[::3, ::5], base[10:11]):
        for block in ("row", "tile"):
            q, t = ops.quantize_fp8(x, block, rows=True, columns=True)
            same(q, _quantize_plain(x.cpu(), block == "tile", E4M3))
            same(t, _quantize_plain(x.cpu().t(), block == "tile", E4M3))


def product_bound(a, b, k):
    return (k / 32 + 1) * 2.0**-22 * (a.abs() @ b.abs().t())


GEMMS = [(1, 1, 1), (1, 300, 128), (5, 7, 129), (128, 128, 128), (256, 256, 512), (256, 256, 640), (130, 260, 1000),
         (257, 513, 1537), (1000, 300, 2048), (512, 1024, 4096), (300, 2500, 384)]


@pytest.mark.parametrize("m,n,k", GEMMS)
@pytest.mark.parametrize("types", [(E4M3, E4M3), (E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)])
def test_gemm(m, n, k, types):
    a, b = rand((m, k), m + k), rand((n, k), n + 7 * k)
    qa, qb = ops.quantize_fp8(a, "row", dtype=types[0])[0], ops.quantize_fp8(b, "tile", dtype=types[1])[0]
    va, vb = qa.dequantize(torch.float64), qb.dequantize(torch.float64)
    want = va @ vb.t()
    got = ops.gemm_fp8(qa, qb, out_dtype=torch.float32)
    _ext.check_status()
    assert bool(((got.double() - want).abs() <= product_bound(va, vb, k)).all())
    bf = ops.gemm_fp8(qa, qb)
    assert bf.dtype == torch.bfloat16 and torch.equal(bf, got.to(torch.bfloat16))


def test_gemm_scales_of_every_block():
    """Each block and row has a scale of its own: codes of one value, scales from 2^-20 to 2^20."""
    g = torch.Generator().manual_seed(9)
    m, n, k = 300, 400, 128 * 11
    ea, eb = (torch.randint(-20, 21, (r, k // 128), generator=g) for r in (m, n))
    a = torch.exp2(ea.float()).repeat_interleave(128, 1).to(torch.bfloat16).cuda()
    b = torch.exp2(eb.float()).repeat_interleave(128, 1).to(torch.bfloat16).cuda()
    qa, qb = ops.quantize_fp8(a)[0], ops.quantize_fp8(b)[0]
    got = ops.gemm_fp8(qa, qb, out_dtype=torch.float32)
    want = a.double() @ b.double().t()
    assert bool(((got.double() - want).abs() <= product_bound(a.double(), b.double(), k)).all())


@pytest.mark.parametrize("m,n,k", [(130, 260, 700), (256, 512, 1024), (700, 77, 300)])
def test_gemm_accumulate_and_strided_output(m, n, k):
    qa, qb = ops.quantize_fp8(rand((m, k), 1))[0], ops.quantize_fp8(rand((n, k), 2))[0]
    va, vb = qa.dequantize(torch.float64), qb.dequantize(torch.float64)
    want = va @ vb.t()
    tol = product_bound(va, vb, k)
    big = torch.full((m + 3, n + 5), 3.0, device="cuda")
    out = big[1:m + 1, 2:n + 2]
    ops.gemm_fp8(qa, qb, out=out, accumulate=True)
    assert bool(((out.double() - want - 3.0).abs() <= tol + 2.0**-23 * (want.abs() + 3)).all())
    ops.gemm_fp8(qa, qb, out=out)
    assert bool(((out.double() - want).abs() <= tol).all())
    out.fill_(3.0)
    assert bool((big == 3.0).all())  # nothing beside the view was written
    bf = torch.full((m, n + 8), 3.0, device="cuda", dtype=torch.bfloat16)
    ops.gemm_fp8(qa, qb, out=bf[:, :n])
    assert torch.equal(bf[:, :n], ops.gemm_fp8(qa, qb)) and bool((bf[:, n:] == 3.0).all())


def test_gemm_not_finite():
    a, b = rand((200, 300), 5), rand((300, 300), 6)
    a[3, 5] = float("nan")
    b[130, 299] = float("inf")
    qa, qb = ops.quantize_fp8(a)[0], ops.quantize_fp8(b)[0]
    got = torch.isnan(ops.gemm_fp8(qa, qb, out_dtype=torch.float32))
    want = torch.zeros_like(got)
    want[3] = True
    want[:, 130] = True
    assert torch.equal(got, want)


def linear64(x, w, dy, grad_dtype=E4M3):
    """The layer from its definition, in 64 bits; also the bounds of its sums."""
    q = lambda t, tile=False, dt=E4M3: _quantize_plain(t.detach().cpu(), tile, dt).dequantize(torch.float64)  # noqa: E731
    xv, wv, xt = q(x), q(w, True), q(x.t())
    dv, dt = q(dy, dt=grad_dtype), q(dy.t(), dt=grad_dtype)
    k, n, t = x.shape[1], w.shape[0], x.shape[0]
    return ((xv @ wv.t(), product_bound(xv, wv, k)), (dv @ wv, product_bound(dv, wv.t(), n)),
            (dt @ xt.t(), product_bound(dt, xt, t)))


def near(got, want, tol, half_step):
    assert bool(((got.cpu().double() - want).abs() <= tol + half_step * (want.abs() + tol)).all())


@pytest.mark.parametrize("t,k,n", [(1, 256, 128), (3, 130, 70), (128, 128, 128), (300, 513, 1025), (640, 1024, 512)])
@pytest.mark.parametrize("grad_dtype", [E4M3, E5M2])
def test_linear(t, k, n, grad_dtype):
    x, w, dy = rand((t, k), 1).requires_grad_(), rand((n, k), 2, spread=0.0).requires_grad_(), rand((t, n), 3)
    y = ops.linear_fp8(x, w, grad_dtype=grad_dtype)
    y.backward(dy)
    for got, (want, tol) in zip((y, x.grad, w.grad), linear64(x, w, dy, grad_dtype)):
        assert got.dtype == torch.bfloat16
        near(got.detach(), want, tol, 2.0**-8)


def test_linear_with_kept_weight_accumulator_and_leading_dimensions():
    x, w, dy = rand((6, 40), 1)[None].expand(2, 6, 40).clone().requires_grad_(), rand((24, 40), 2), rand((12, 24), 3)
    acc = torch.ones(24, 40, device="cuda")
    w._mvp_grad_acc = acc
    w8 = ops.quantize_fp8(w, "tile", rows=True, columns=True)
    y = ops.linear_fp8(x, w, w8)
    assert y.shape == (2, 6, 24)
    y.backward(dy.view(2, 6, 24))
    (wy, ty), (wx, tx), (ww, tw) = linear64(x.detach().view(12, 40), w, dy)
    near(y.detach().view(12, 24), wy, ty, 2.0**-8)
    near(x.grad.view(12, 40), wx, tx, 2.0**-8)
    near(acc, ww + 1, tw, 2.0**-23)
    assert w.grad is None
    y2 = ops.linear_fp8(x, w)  # the same product without the kept weight
    assert torch.equal(y2, y)
    (y2.sum() * 0).backward()  # an expanded gradient


@pytest.mark.parametrize("need", [(True, False), (False, True)])
def test_linear_one_gradient(need):
    x, w, dy = rand((70, 200), 1).requires_grad_(need[0]), rand((90, 200), 2).requires_grad_(need[1]), rand((70, 90), 3)
    ops.linear_fp8(x, w).backward(dy)
    _, dx, dw = linear64(x, w, dy)
    if need[0]:
        near(x.grad, *dx, 2.0**-8)
        assert w.grad is None
    else:
        near(w.grad, *dw, 2.0**-8)
        assert x.grad is None


def test_linear_gradient_against_differences():
    """The gradient of a smooth loss against differences of the unquantised layer: as close as 8-bit operands allow (half
    a step is 2^-4 of a value; over 128 and more terms the relative error of a sum is below it)."""
    x, w, r = rand((64, 256), 1, spread=0.0), rand((128, 256), 2, spread=0.0) * 0.1, rand((64, 128), 3, spread=0.0)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    (ops.linear_fp8(xr, wr).float() * r.float()).sum().backward()
    loss = lambda a, b: float(((a.double() @ b.double().t()) * r.double()).sum())  # noqa: E731
    for grad, base, f in ((xr.grad, x, lambda v: loss(v, w)), (wr.grad, w, lambda v: loss(x, v))):
        d = grad.double() / grad.double().norm()
        eps = 1e-3
        diff = (f(base.double() + eps * d) - f(base.double() - eps * d)) / (2 * eps)
        assert abs(diff - float(grad.double().norm())) <= 2.0**-4 * abs(diff)


def test_linear_strided_operands():
    """Weights and inputs that are slices or transposes of larger tensors."""
    big, wide = rand((140, 600), 1), rand((500, 301), 2, spread=0.0)
    for x, w in ((big[3:133:2, 7:307], wide[:90].t()[:300].t()), (big.t()[5:65], wide[:140].t()[10:50]),
                 (big[:, :301][:1], wide[::4])):
        x = x[:, : min(x.shape[1], w.shape[1])]
        w = w[:, : x.shape[1]]
        got = ops.linear_fp8(x, w)
        assert torch.equal(got, ops.linear_fp8(x.contiguous(), w.contiguous()))


def test_linear_on_one_dimension_and_tokens_of_every_count():
    w = rand((40, 72), 2, spread=0.0)
    x = rand((300, 72), 1)
    full = ops.linear_fp8(x, w)
    assert torch.equal(ops.linear_fp8(x[5], w), full[5])
    for t in (1, 2, 31, 127, 129, 255, 257):  # a row's blocks are its own: its result does not depend on the others
        assert torch.equal(ops.linear_fp8(x[:t], w), full[:t])


def test_linear_empty_and_no_grad():
    w = rand((32, 64), 2).requires_grad_()
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = ops.linear_fp8(x, w)
    assert y.shape == (0, 32)
    y.sum().backward()
    assert x.grad.shape == (0, 64)
    with torch.no_grad():
        assert not ops.linear_fp8(rand((4, 64)), w).requires_grad


def test_linear_other_stream_and_graph():
    x, w = rand((200, 384), 1), rand((300, 384), 2)
    want = ops.linear_fp8(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.linear_fp8(x, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        out = ops.linear_fp8(x, w)
    for seed in (5, 6):
        x.copy_(rand((200, 384), seed))
        g.replay()
        assert torch.equal(out, ops.linear_fp8(x, w))


def test_calls_on_two_streams_at_once():
    """Layers and updates under way together: each call has its own workspace, results are those of calls alone."""
    x, w, dy = rand((700, 900), 1), rand((1100, 900), 2), rand((700, 1100), 3)
    u = torch.randn(3, 200, 600, device="cuda", generator=torch.Generator("cuda").manual_seed(4))

    def layer():
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = ops.linear_fp8(a, b)
        return (y.detach(), *torch.autograd.grad(y, (a, b), dy))

    want_l, want_o = layer(), ops.orthogonalize(u)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            got[0].append(layer())
        with torch.cuda.stream(streams[1]):
            got[1].append(ops.orthogonalize(u))
            got[1].append(ops.linear_fp8(x, w))
    torch.cuda.synchronize()
    _ext.check_status()
    for r in got[0]:
        assert all(torch.equal(a, b) for a, b in zip(r, want_l))
    for i, r in enumerate(got[1]):
        assert torch.equal(r, want_o if i % 2 == 0 else want_l[0])


def test_offsets_past_32_bits():
    """More than 2^31 values in, codes out and products out: the far end equals the same rows by themselves."""
    rows, cols = 65600, 33000
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    tail = rand((200, cols), 1)
    x[:-200] = 1.0
    x[-200:] = tail
    q, t = ops.quantize_fp8(x, columns=True)
    alone = ops.quantize_fp8(tail)[0]
    assert torch.equal(q.data[-200:].view(torch.uint8), alone.data.view(torch.uint8))
    assert torch.equal(q.exponents()[-200:], alone.exponents())
    # the last whole column block is rows 65408 .. 65535, the rest of the matrix ends within the next
    part = ops.quantize_fp8(x[65408:], rows=False, columns=True)[1]
    assert torch.equal(t.data[:, 65408:].contiguous().view(torch.uint8), part.data.view(torch.uint8))
    del x, q, t
    a, b = rand((46400, 128), 2), rand((46400, 128), 3)
    qa, qb = ops.quantize_fp8(a)[0], ops.quantize_fp8(b)[0]
    y = ops.gemm_fp8(qa, qb)
    small = ops.gemm_fp8(ops.quantize_fp8(a[-300:])[0], qb)
    assert torch.equal(y[-300:], small)


def test_refusals():
    x, w = rand((4, 64)), rand((8, 64))
    with pytest.raises(TypeError):
        ops.linear_fp8(x, w.float())
    with pytest.raises(ValueError):
        ops.linear_fp8(x, w.cpu())
    with pytest.raises(ValueError):
        ops.linear_fp8(x, w, ops.quantize_fp8(w.cpu(), "tile", rows=True, columns=True))
    q = ops.quantize_fp8(x)[0]
    with pytest.raises(ValueError):
        ops.gemm_fp8(q, ops.quantize_fp8(w.cpu())[0])
    with pytest.raises((RuntimeError, ValueError)):  # an output whose rows overlap
        ops.gemm_fp8(q, q, out=torch.empty(4, device="cuda")[None].expand(4, 4))
    with pytest.raises((RuntimeError, ValueError)):  # no unit column stride
        ops.gemm_fp8(q, q, out=torch.empty(4, 4, device="cuda").t()[:, :])
    short = ops.Fp8Matrix(q.data, q.scale[:, :, :16].contiguous(), q.cols)
    with pytest.raises(RuntimeError):
        ops.gemm_fp8(short, q)
