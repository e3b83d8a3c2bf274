"""Adapters that no row uses: their gradients are zero whatever they and their factors hold."""
import pytest
import torch

import mlx_kquant_b200 as kq
from test_lora_gpu import TYPES, made

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("factor", [float("inf"), float("nan")])
@pytest.mark.parametrize("T", [7, 2500])
@pytest.mark.parametrize("dt,pt", TYPES)
def test_factor_of_an_unused_adapter(dt, pt, T, factor):
    y, x, a, b, s, dy = made(2, T, 72, 40, 8, 3, dt, pt)
    ids = torch.arange(T, dtype=torch.int32, device="cuda") % 2 * 2      # 0 and 2
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    want = torch.autograd.grad(kq.lora_update(y, *leaves, ids, s), leaves, dy)
    s[1] = factor
    a[1], b[1] = factor, factor
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    out = kq.lora_update(y, *leaves, ids, s)
    got = torch.autograd.grad(out, leaves, dy)
    assert out.isfinite().all() and not got[1][1].any() and not got[2][1].any()
    for p, q in zip(want, got):
        assert torch.equal(p, q)
