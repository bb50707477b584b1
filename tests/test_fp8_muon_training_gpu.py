"""8-bit linear layers and Muon in the training runtime on the GPU: a decoder step, the flat optimizer's update, and a layer
with its update, against the formulas in 64 bits."""

import math

import pytest
import torch

from mvp_engine import ops
from mvp_engine.models.qwen3 import build_qwen3
from mvp_engine.ops import _ext
from mvp_engine.ops.fp8 import _quantize_plain
from mvp_engine.parallel.fsdp import NativeFSDP
from mvp_engine.parallel.optim import FlatMuon, is_hidden_matrix

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

TINY = dict(vocab_size=512, hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2)
NS_TOL = 3e-3  # documented for the iteration


def ns64(u):
    x = u.double() / max(float(u.double().norm()), 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(5):
        s = x @ x.T
        x = 3.4445 * x + (-4.775 * s + 2.0315 * s @ s) @ x
    return x.T if tall else x


def runtime(precision, ckpt=False):
    model = build_qwen3("mvp/qwen3-tiny", seed=3, device="meta", **TINY)
    model.set_linear_precision(precision)
    if ckpt:
        model.gradient_checkpointing_enable()
    fsdp = NativeFSDP(model, group=None, device=torch.device("cuda"), param_dtype=torch.bfloat16)
    fsdp.train()
    return fsdp


def backward(fsdp, seed=1):
    x = torch.randint(0, 512, (1, 300), generator=torch.Generator().manual_seed(seed)).cuda()
    loss = fsdp(input_ids=x, labels=x)["loss"].sum() / 299
    loss.backward()
    return float(loss.detach())


def grads(fsdp):
    return {e.fqns[0]: u.grad[e.offset:e.offset + e.numel].view(e.shape).clone()
            for u in fsdp.units if u.trainable for e in u.entries}


def test_decoder_gradients_with_8bit_products():
    got = {}
    for precision in ("bf16", "fp8"):
        fsdp = runtime(precision)
        loss = backward(fsdp)
        fsdp.finish_grad_sync()
        got[precision] = (loss, grads(fsdp))
        _ext.check_status()
    # an e4m3 operand is off by 2^-4 of a value at most and 2^-5 / sqrt(3) of it on average: 0.026 for a product of two
    assert abs(got["fp8"][0] - got["bf16"][0]) <= 0.05 * got["bf16"][0]
    for n, g in got["bf16"][1].items():
        h = got["fp8"][1][n]
        cos = float((g.double() * h.double()).sum() / (g.double().norm() * h.double().norm()))
        assert cos > 0.95, (n, cos)
    layer = "model.layers.0.self_attn.q_proj.weight"
    assert not torch.equal(got["bf16"][1][layer], got["fp8"][1][layer])


@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_flat_muon_step(precision):
    """Two steps: masters, momenta and bf16 weights of every hidden matrix follow the formulas."""
    fsdp = runtime(precision, ckpt=precision == "fp8")
    opt = FlatMuon(fsdp, lr=1e-2, momentum=0.9)
    for step in range(2):
        backward(fsdp, step)
        norm = float(fsdp.clip_grad_norm_(0.5))
        clip = min(1.0, 0.5 / (norm + 1e-6))
        want = {}
        for u in fsdp.units:
            for e in u.entries:
                if not is_hidden_matrix(e.fqns[0], e.shape):
                    continue
                at = slice(e.offset, e.offset + e.numel)
                g, m, p = (t[at].view(e.shape).double() for t in (u.grad, u.exp_avg, u.master.data))
                g = g * clip
                m = m + 0.1 * (g - m)
                delta = 1e-2 * 0.2 * math.sqrt(max(e.shape)) * ns64(g + 0.9 * (m - g))
                want[e.fqns[0]] = (p * (1 - 1e-2 * 0.1) - delta, m, delta)
        assert len(want) == 14
        opt.step()
        torch.cuda.synchronize()
        _ext.check_status()
        for u in fsdp.units:
            for e in u.entries:
                if e.fqns[0] not in want:
                    continue
                at = slice(e.offset, e.offset + e.numel)
                p, m, delta = want[e.fqns[0]]
                got = u.master.data[at].view(e.shape)
                assert float((got.double() - p).norm()) <= NS_TOL * float(delta.norm()) + 2.0**-22 * float(p.norm())
                # the clip coefficient is read back from a 32-bit norm, then four roundings
                assert float((u.exp_avg[at].view(e.shape).double() - m).norm()) <= 1e-6 * float(m.norm())
                assert torch.equal(u.full[at].view(e.shape), got.to(torch.bfloat16))


def test_layer_and_update_together():
    """y = Q(x) Q(w)^T, its weight gradient into the accumulator, the Muon step that consumes it and writes the weights that
    the next product quantises: two steps against the formulas."""
    g = torch.Generator().manual_seed(7)
    rows, cols, tokens = 300, 520, 250
    p = (torch.randn(rows, cols, generator=g) * 0.05).cuda()
    w, acc, m = p.to(torch.bfloat16), torch.zeros(rows, cols, device="cuda"), torch.zeros(rows, cols, device="cuda")
    w._mvp_grad_acc = acc
    q = lambda t, tile=False: _quantize_plain(t.detach().float().cpu(), tile, torch.float8_e4m3fn).dequantize(torch.float64)  # noqa: E731
    for _ in range(2):
        x = torch.randn(tokens, cols, generator=g).to(torch.bfloat16).cuda().requires_grad_()
        dy = torch.randn(tokens, rows, generator=g).to(torch.bfloat16).cuda()
        y = ops.linear_fp8(x, w)
        want = q(x) @ q(w, True).t()
        bound = (cols / 32 + 1) * 2.0**-22 * (q(x).abs() @ q(w, True).abs().t())
        assert bool(((y.detach().cpu().double() - want).abs() <= bound + 2.0**-8 * (want.abs() + bound)).all())
        y.backward(dy)
        dt, xt = q(dy.t()), q(x.t())
        dw, bound = dt @ xt.t(), (tokens / 32 + 1) * 2.0**-22 * (dt.abs() @ xt.abs().t())
        assert bool(((acc.cpu().double() - dw).abs() <= bound + 2.0**-23 * dw.abs()).all())
        gr, m64 = acc.double(), m.double()
        m64 = m64 + 0.1 * (gr - m64)
        delta = 0.02 * ns64(gr + 0.9 * (m64 - gr))
        after = p.double() * (1 - 0.02 * 0.1) - delta
        ops.muon_step_(p, acc, m, lr=0.02, momentum=0.9, p_bf16=w)
        assert float((p.double() - after).norm()) <= NS_TOL * float(delta.norm()) + 2.0**-22 * float(after.norm())
        assert torch.equal(w, p.to(torch.bfloat16))
        acc.zero_()
    _ext.check_status()


def test_step_captured_into_a_graph():
    """Forward, backward and update of a layer in one graph: replays equal eager steps bit for bit."""
    g = torch.Generator().manual_seed(11)
    rows, cols, tokens = 256, 384, 200
    x = torch.randn(tokens, cols, generator=g).to(torch.bfloat16).cuda()
    dy = torch.randn(tokens, rows, generator=g).to(torch.bfloat16).cuda()
    start = (torch.randn(rows, cols, generator=g) * 0.05).cuda()

    def fresh():
        p = start.clone()
        return p, p.to(torch.bfloat16), torch.zeros_like(p), torch.zeros_like(p)

    def step(p, w, acc, m):
        w._mvp_grad_acc = acc
        xg = x.detach().requires_grad_()
        ops.linear_fp8(xg, w).backward(dy)
        ops.muon_step_(p, acc, m, lr=0.02, p_bf16=w)
        acc.zero_()
        return xg.grad

    eager = fresh()
    for _ in range(3):
        want = step(*eager)
    torch.cuda.synchronize()
    state = fresh()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        warm = fresh()
        step(*warm)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*state)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(eager, state):
        assert torch.equal(a, b)
    assert torch.equal(got, want)
