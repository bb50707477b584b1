"""8-bit blocks on the CPU path: the format from its definition, the linear layer, and what is refused."""

import math

import pytest
import torch

from mvp_engine import ops

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
TOP = {E4M3: 448.0, E5M2: 57344.0}
MANTISSA = {E4M3: (3, -6), E5M2: (2, -14)}


def code_of(v, dtype):
    """The nearest 8-bit value, ties to even, from the type's definition."""
    bits, low = MANTISSA[dtype]
    if v == 0:
        return 0.0
    step = 2.0 ** (max(math.floor(math.log2(abs(v))), low) - bits)
    return round(v / step) * step  # Python rounds halves to even


def block_of(values, dtype):
    amax = max(abs(v) for v in values)
    e = -127
    while amax > TOP[dtype] * 2.0**e:
        e += 1
    return [code_of(v / 2.0**e, dtype) for v in values], e


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("shape", [(3, 5), (2, 130), (130, 2)])
def test_format_from_its_definition(shape, dtype):
    x = (torch.randn(shape, generator=torch.Generator().manual_seed(1)) * 3).to(torch.bfloat16)
    x[0, 0], x[0, 1] = TOP[dtype], 2.0**-30
    q, t = ops.quantize_fp8(x, rows=True, columns=True, dtype=dtype)
    for m, v in ((q, x), (t, x.t())):
        assert m.shape == tuple(v.shape)
        assert m.data.shape == (v.shape[0], -(-v.shape[1] // 128) * 128)
        codes, exps = m.data.float(), m.exponents()
        for r in range(v.shape[0]):
            for b in range(exps.shape[1]):
                want, e = block_of(v[r, b * 128:(b + 1) * 128].tolist(), dtype)
                assert int(exps[r, b]) == e
                assert codes[r, b * 128:b * 128 + len(want)].tolist() == want
        assert bool((codes[:, v.shape[1]:] == 0).all())
        torch.testing.assert_close(m.dequantize(), (codes.view(v.shape[0], -1, 128) * torch.exp2(exps.float())[..., None])
                                   .view(v.shape[0], -1)[:, :v.shape[1]], rtol=0, atol=0)


def test_tiles_share_scales_between_both_orientations():
    x = torch.randn(300, 260, generator=torch.Generator().manual_seed(2))
    q, t = ops.quantize_fp8(x, "tile", rows=True, columns=True)
    torch.testing.assert_close(q.dequantize(), t.dequantize().t(), rtol=0, atol=0)
    e = q.exponents()
    assert e.shape == (300, 3) and bool((e[:128] == e[0]).all()) and bool((e[256:] == e[256]).all())
    for i in range(3):
        for j in range(3):
            amax = float(x[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].abs().max())
            assert 448 * 2.0 ** (int(e[i * 128, j]) - 1) < amax <= 448 * 2.0 ** int(e[i * 128, j])


def test_zero_tiny_and_not_finite_blocks():
    x = torch.zeros(4, 256)
    x[1, 0], x[2, 200], x[3, 3] = 1e-40, float("inf"), float("nan")
    q = ops.quantize_fp8(x)[0]
    assert q.exponents().tolist() == [[-127, -127], [-127, -127], [-127, 0], [0, -127]]
    v = q.dequantize()
    assert bool((v[0] == 0).all()) and 0 < float(v[1, 0]) < 1.1e-40
    assert torch.isnan(v[2, 128:]).all() and bool((v[2, :128] == 0).all())
    assert torch.isnan(v[3, :128]).all() and bool((v[3, 128:] == 0).all())


def test_rounding_is_within_half_a_step():
    x = torch.randn(64, 512, generator=torch.Generator().manual_seed(3))
    for dtype in (E4M3, E5M2):
        m = ops.quantize_fp8(x, dtype=dtype)[0]
        v, scale = m.dequantize(), torch.exp2(m.exponents().float()).repeat_interleave(128, 1)
        bits, low = MANTISSA[dtype]
        assert bool(((v - x).abs() <= x.abs() * 2.0 ** -(bits + 1) + scale * 2.0 ** (low - bits - 1)).all())


@pytest.mark.parametrize("grad_dtype", [E4M3, E5M2])
def test_linear_and_gradients(grad_dtype):
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn(2, 9, 150, generator=g).requires_grad_(), torch.randn(70, 150, generator=g).requires_grad_()
    dy = torch.randn(2, 9, 70, generator=g)
    y = ops.linear_fp8(x, w, grad_dtype=grad_dtype)
    y.backward(dy)
    x2, d2 = x.detach().view(18, 150), dy.view(18, 70)
    q = lambda t, block="row", dt=E4M3: ops.quantize_fp8(t, block, dtype=dt)[0].dequantize(torch.float64)  # noqa: E731
    wv = q(w, "tile")
    want = (q(x2) @ wv.t(), q(d2, dt=grad_dtype) @ wv, q(d2.t(), dt=grad_dtype) @ q(x2.t()).t())
    for got, ref in zip((y.view(18, 70), x.grad.view(18, 150), w.grad), want):
        # 32-bit sums of at most 150 products
        torch.testing.assert_close(got.detach().double(), ref, rtol=1e-5, atol=150 * 2.0**-24 * float(ref.abs().max()) + 1e-5)


def test_linear_kept_weight_and_accumulator():
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(5, 40, generator=g).requires_grad_(), torch.randn(30, 40, generator=g)
    w._mvp_grad_acc = torch.ones(30, 40)
    y = ops.linear_fp8(x, w, ops.quantize_fp8(w, "tile", rows=True, columns=True))
    assert torch.equal(y, ops.linear_fp8(x, w))
    y.sum().backward()
    plain = w.clone().requires_grad_()
    ops.linear_fp8(x, plain).sum().backward()
    torch.testing.assert_close(w._mvp_grad_acc, plain.grad + 1, rtol=1e-6, atol=1e-6)


def test_linear_twice_differentiated_is_refused():
    x = torch.randn(3, 8, requires_grad=True)
    (gx,) = torch.autograd.grad(ops.linear_fp8(x, torch.randn(4, 8)).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_refusals():
    x, w = torch.randn(4, 8), torch.randn(6, 8)
    for bad in (lambda: ops.quantize_fp8(x, "column"), lambda: ops.quantize_fp8(x[0]),
                lambda: ops.quantize_fp8(x, rows=False), lambda: ops.quantize_fp8(torch.empty(0, 8)),
                lambda: ops.linear_fp8(x, torch.randn(6, 9)), lambda: ops.linear_fp8(x, w[0]),
                lambda: ops.linear_fp8(x, w, (None, None)),
                lambda: ops.linear_fp8(x, w, ops.quantize_fp8(x, "tile", rows=True, columns=True))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.quantize_fp8(x, dtype=torch.int8), lambda: ops.quantize_fp8(x.double()),
                lambda: ops.linear_fp8(x, w, grad_dtype=torch.bfloat16), lambda: ops.gemm_fp8(x, w)):
        with pytest.raises(TypeError):
            bad()
    q, r = ops.quantize_fp8(x)[0], ops.quantize_fp8(torch.randn(4, 9))[0]
    with pytest.raises(ValueError):
        ops.gemm_fp8(q, r)
    with pytest.raises(ValueError):
        ops.gemm_fp8(q, q, accumulate=True)
    with pytest.raises(ValueError):
        ops.gemm_fp8(q, q, out=torch.zeros(4, 4, dtype=torch.bfloat16), accumulate=True)
    with pytest.raises(ValueError):
        ops.gemm_fp8(q, q, out=torch.zeros(4, 5))
    with pytest.raises(TypeError):
        ops.gemm_fp8(q, q, out_dtype=torch.float16)
    acc = torch.randn(6, 8)
    acc._mvp_grad_acc = torch.zeros(6, 7)
    with pytest.raises(ValueError):
        ops.linear_fp8(x.requires_grad_(), acc)
