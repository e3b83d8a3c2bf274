"""Low-rank adapters on the quantized layers, and a routed layer of all of them, against float64 on the dequantized weights."""
import numpy as np
import pytest
import torch

import mlx_kquant_b200 as kq
from gpu_util import mint_wire
from mlx_kquant_b200.moe import combine, moe_router_grouped, swiglu
from mlx_kquant_b200.nn import KQuantLinear, KQuantLoRALinear, KQuantLoRASwitchLinear, KQuantSwitchLinear

pytestmark = pytest.mark.gpu


def wire(codec, *shape, seed):
    rng = np.random.default_rng(seed)
    w = rng.normal(0, shape[-1] ** -0.5, shape).astype(np.float32)
    flat = mint_wire(codec, w.reshape(-1, shape[-1]))
    return torch.from_numpy(flat.reshape(*shape[:-1], -1)).cuda()


def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def linear(bias, codec="q4_k", N=96, K=512, **kw):
    base = KQuantLinear(K, N, bias, codec).cuda()
    base.weight.copy_(wire(codec, N, K, seed=1))
    if bias:
        base.bias.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    layer = KQuantLoRALinear(base, **kw)
    g = torch.Generator(device="cuda").manual_seed(2)
    with torch.no_grad():
        layer.lora_b.copy_(torch.randn(layer.lora_b.shape, device="cuda", generator=g) * 0.1)
        layer.scaling.copy_(torch.rand(layer.scaling.shape, device="cuda", generator=g) + 0.5)
    return layer


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("T", [1, 5, 40])
def test_linear(bias, T):
    layer = linear(bias, rank=8, n_adapters=3, codec="q8_0" if bias else "q4_k")
    base = layer.base
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, 512, device="cuda", generator=g).bfloat16().requires_grad_()
    ids = torch.randint(-1, 3, (T,), device="cuda", generator=g, dtype=torch.int32)
    y = layer(x, ids)
    W = kq.dequantize(base.weight, base.scales, base.kquant_type, torch.float32).double()
    xd = x.detach().double().requires_grad_()
    A, B = layer.lora_a.detach().double().requires_grad_(), layer.lora_b.detach().double().requires_grad_()
    on = (ids >= 0).double() * layer.scaling.double()[ids.clamp(min=0).long()]
    at = ids.clamp(min=0).long()
    ref = xd @ W.T + (base.bias.double() if bias else 0.0) + on[:, None] * torch.einsum("tnr,trk,tk->tn", B[at], A[at], xd)
    dy = torch.randn(T, 96, device="cuda", generator=g).bfloat16()
    got = torch.autograd.grad(y, (x, layer.lora_a, layer.lora_b), dy)
    want = torch.autograd.grad(ref, (xd, A, B), dy.double())
    # y: the product, the bias and the update are rounded to bf16 one after another (2^-9 rms each at most); dx the same
    assert off(y, ref) < 3 * 2.0 ** -9 + 2e-3 and off(got[0], want[0]) < 2 * 2.0 ** -9 + 2e-3
    assert off(got[1], want[1]) < 1e-5 and off(got[2], want[2]) < 1e-5
    with torch.no_grad():
        assert off(layer(x, ids), ref.detach()) < 3 * 2.0 ** -9 + 2e-3
        if not bias:
            plain = kq.quantized_matmul_lora(x.detach(), base.weight, base.scales, base.kquant_type, layer.lora_a, layer.lora_b, ids,
                                             layer.scaling)
            assert torch.equal(plain, layer(x, ids))
            side = torch.cuda.Stream()
            again = kq.quantized_matmul_lora(x.detach(), base.weight, base.scales, base.kquant_type, layer.lora_a, layer.lora_b, ids,
                                             layer.scaling, stream=side)
            torch.cuda.synchronize()
            assert torch.equal(again, plain)
    if not bias:
        y2 = kq.quantized_matmul_lora(x, base.weight, base.scales, base.kquant_type, layer.lora_a, layer.lora_b, ids, layer.scaling)
        assert torch.equal(y2, y.detach())
        for p, q in zip(torch.autograd.grad(y2, (x, layer.lora_a, layer.lora_b), dy), got):
            assert torch.equal(p, q)


def test_float32_rows_and_a_step():
    layer = linear(False, rank=4)
    x = torch.randn(6, 512, device="cuda", requires_grad=True)
    opt = torch.optim.SGD(layer.parameters(), lr=0.1)
    before = layer.lora_a.detach().clone()
    y = layer(x)
    assert y.dtype == torch.bfloat16
    y.float().square().sum().backward()
    assert x.grad.dtype == torch.float32 and torch.isfinite(x.grad).all()
    opt.step()
    assert not torch.equal(before, layer.lora_a) and layer.base.weight.grad is None


@pytest.mark.parametrize("form", ["token", "slot", "flat"])
def test_switch_linear(form):
    E, N, K, T, R, G = 6, 72, 256, 9, 3, 2
    base = KQuantSwitchLinear(E, N, K, False, "q4_k").cuda()
    base.weight.copy_(wire("q4_k", E, N, K, seed=3))
    layer = KQuantLoRASwitchLinear(base, 8, G, 0.75)
    g = torch.Generator(device="cuda").manual_seed(4)
    with torch.no_grad():
        layer.lora_b.copy_(torch.randn(layer.lora_b.shape, device="cuda", generator=g) * 0.1)
    idx = torch.randint(0, E, (T, R), device="cuda", generator=g, dtype=torch.int32)
    ids = torch.randint(0, G, (T,), device="cuda", generator=g, dtype=torch.int32)
    x = torch.randn(T, 1 if form == "token" else R, 1, K, device="cuda", generator=g).half()
    if form == "flat":
        x, idx, ids = x.reshape(T * R, 1, K), idx.reshape(-1), ids.repeat_interleave(R)
    x.requires_grad_()
    y = layer(x, idx, ids)
    W = kq.dequantize(base.weight, base.scales, "q4_k", torch.float32).double()
    xd = x.detach().double().requires_grad_()
    A, B = layer.lora_a.detach().double().requires_grad_(), layer.lora_b.detach().double().requires_grad_()
    rows = xd.expand(T, R, 1, K).reshape(-1, K) if form == "token" else xd.reshape(-1, K)
    e = idx.reshape(-1).long()
    a = ids.long() if form == "flat" else ids.long().repeat_interleave(R)
    ref = torch.einsum("tnk,tk->tn", W[e], rows) + 0.75 * torch.einsum("tnr,trk,tk->tn", B[a, e], A[a, e], rows)
    assert off(y.reshape(-1, N), ref) < 2 * 2.0 ** -12 + 2e-3
    dy = torch.randn(y.shape, device="cuda", generator=g).half()
    got = torch.autograd.grad(y, (x, layer.lora_a, layer.lora_b), dy)
    want = torch.autograd.grad(ref, (xd, A, B), dy.double().reshape(-1, N))
    assert off(got[0], want[0]) < 2 * 2.0 ** -12 + 2e-3
    assert off(got[1], want[1]) < 1e-5 and off(got[2], want[2]) < 1e-5
    with torch.no_grad():
        assert torch.equal(layer(x, idx, ids), y.detach())


def test_switch_linear_refuses_other_shapes():
    layer = KQuantLoRASwitchLinear(KQuantSwitchLinear(4, 8, 256, False, "q4_k").cuda(), 2)
    with pytest.raises(ValueError, match="x must be"):
        layer(torch.zeros(3, 2, 256, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"))


def test_routed_layer_with_adapters():
    """A mixture-of-experts layer as an adapted model runs it: router, gate | up and down products with adapters of two requests, the
    weighted sum - forward, gradients of the router's logits and of all adapters, and the same forward from a graph."""
    T, E, R, H, F, G = 24, 8, 2, 256, 256, 2
    gu = KQuantSwitchLinear(E, 2 * F, H, False, "q4_k").cuda()
    dn = KQuantSwitchLinear(E, H, F, False, "q4_k").cuda()
    gu.weight.copy_(wire("q4_k", E, 2 * F, H, seed=5))
    dn.weight.copy_(wire("q4_k", E, H, F, seed=6))
    up, down = KQuantLoRASwitchLinear(gu, 8, G), KQuantLoRASwitchLinear(dn, 4, G)
    g = torch.Generator(device="cuda").manual_seed(7)
    for m in (up, down):
        with torch.no_grad():
            m.lora_b.copy_(torch.randn(m.lora_b.shape, device="cuda", generator=g) * 0.1)
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16().requires_grad_()
    logits = torch.randn(T, E, device="cuda", generator=g).requires_grad_()
    bias = torch.randn(E, device="cuda", generator=g) * 0.1
    ids = torch.randint(0, G, (T,), device="cuda", generator=g, dtype=torch.int32)

    def layer(kernels):
        idx, w = moe_router_grouped(logits, R, 4, 2, bias=bias, scale=1.5)
        h = up(x.view(T, 1, 1, H), idx, ids).view(T * R, 2 * F)
        h = swiglu(h[:, :F], h[:, F:]) if kernels else (torch.nn.functional.silu(h[:, :F].float()) * h[:, F:].float()).bfloat16()
        d = down(h.view(T, R, 1, F), idx, ids).view(T * R, H)
        return combine(d, w, R) if kernels else (d.view(T, R, H).float() * w[:, :, None]).sum(1)

    y = layer(False)
    dy = torch.randn(T, H, device="cuda", generator=g)
    leaves = (logits, x, up.lora_a, up.lora_b, down.lora_a, down.lora_b)
    got = torch.autograd.grad(y, leaves, dy)
    # the same in float64
    Wu, Wd = (kq.dequantize(m.weight, m.scales, "q4_k", torch.float32).double() for m in (gu, dn))
    ld, xd, ua, ub, da, db = (t.detach().double().requires_grad_() for t in leaves)
    idx = moe_router_grouped(logits.detach(), R, 4, 2, bias=bias)[0].long()
    s = torch.sigmoid(ld).gather(1, idx)
    w = 1.5 * s / s.sum(1, keepdim=True)
    e, a = idx.reshape(-1), ids.long().repeat_interleave(R)
    rows = xd.repeat_interleave(R, 0)
    h = torch.einsum("tnk,tk->tn", Wu[e], rows) + torch.einsum("tnr,trk,tk->tn", ub[a, e], ua[a, e], rows)
    h = torch.nn.functional.silu(h[:, :F]) * h[:, F:]
    d = torch.einsum("tnk,tk->tn", Wd[e], h) + torch.einsum("tnr,trk,tk->tn", db[a, e], da[a, e], h)
    ref = (d.view(T, R, H) * w[:, :, None]).sum(1)
    want = torch.autograd.grad(ref, (ld, xd, ua, ub, da, db), dy.double())
    # bf16 between the steps: five roundings forward, as many back, 2^-9 rms each at most
    assert off(y, ref) < 5 * 2.0 ** -9 + 2e-3
    for p, q in zip(got, want):
        assert off(p, q) < 10 * 2.0 ** -9 + 2e-3
    with torch.no_grad():
        eager = layer(True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(True)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(True)
        graph.replay()
        assert torch.equal(out, eager) and off(eager, ref.detach()) < 6 * 2.0 ** -9 + 2e-3
