"""Forward-mode differentiation: what has no rule for it refuses, rather than leave the tangent out."""
import pytest
import torch
from torch.autograd import forward_ad

import mlx_kquant_b200 as kq
from mlx_kquant_b200 import lora, moe

gpu = pytest.param("cuda", marks=pytest.mark.gpu)


@pytest.fixture(params=[True, False], ids=["front", "python"])
def path(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(lora, "_front_lora", lambda *a: None)
        monkeypatch.setattr(moe, "_front_route", lambda *a: None)


@pytest.mark.parametrize("device", ["cpu", gpu])
@pytest.mark.parametrize("which", range(5))
def test_low_rank_updates(path, device, which):
    z = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device=device)  # noqa: E731
    ids = torch.zeros(4, dtype=torch.int32, device=device)
    idx = torch.zeros(4, 2, dtype=torch.int32, device=device)
    with forward_ad.dual_level():
        for op, args, rest in ((kq.lora_update, [z(4, 6), z(4, 8), z(2, 3, 8), z(2, 6, 3), torch.ones(2, device=device)], (ids,)),
                               (moe.gather_lora_update, [z(4, 2, 6), z(4, 8), z(2, 5, 3, 8), z(2, 5, 6, 3), torch.ones(2, device=device)], (idx, ids))):
            args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises((ValueError, RuntimeError), match="forward-mode"):
                op(*args[:4], *rest, args[4])


@pytest.mark.gpu
@pytest.mark.parametrize("needs", [False, True])
def test_router(path, needs):
    x = torch.randn(3, 16, device="cuda", requires_grad=needs)
    with forward_ad.dual_level():
        with pytest.raises((ValueError, RuntimeError), match="forward-mode|forward mode|jvp"):
            moe.moe_router_grouped(forward_ad.make_dual(x, torch.ones_like(x)), 2)
    assert moe.moe_router_grouped(x, 2)[0].shape == (3, 2)


@pytest.mark.gpu
def test_composed_product():
    w = torch.zeros(8, 144, dtype=torch.uint8, device="cuda")
    x = torch.ones(2, 256, dtype=torch.bfloat16, device="cuda")
    a, b = torch.ones(1, 2, 256, dtype=torch.bfloat16, device="cuda"), torch.ones(1, 8, 2, dtype=torch.bfloat16, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises((ValueError, RuntimeError), match="forward-mode"):
            kq.quantized_matmul_lora(forward_ad.make_dual(x, torch.ones_like(x)), w, None, "q4_k", a, b)


def test_host_router_has_tangents():
    x, dx = torch.randn(3, 16, dtype=torch.float64).float(), torch.randn(3, 16)
    with forward_ad.dual_level():
        _, w = moe.moe_router_grouped(forward_ad.make_dual(x, dx), 2)
        tangent = forward_ad.unpack_dual(w).tangent
    leaf = x.clone().requires_grad_()
    _, w = moe.moe_router_grouped(leaf, 2)
    g = torch.randn_like(w)
    dl, = torch.autograd.grad(w, leaf, g)
    torch.testing.assert_close((tangent * g).sum(), (dl * dx).sum(), rtol=1e-4, atol=1e-5)
