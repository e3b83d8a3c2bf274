"""moe_router_grouped where some groups have one available expert and others more: a group's sum runs over those that it has."""
import numpy as np
import pytest
import torch

from gpu_util import TORCH_DT
from mlx_kquant_b200.moe import moe_router_grouped
from route_plain import route

pytestmark = pytest.mark.gpu


def masked(T, E, groups, seed):
    """Logits whose groups have none, one, two or all of their experts, by turns of chance."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, groups, E // groups, generator=g) * 1.5
    order = torch.rand(x.shape, generator=g).argsort(dim=2).argsort(dim=2)
    there = torch.tensor([0, 1, 1, 2, E])[torch.randint(0, 5, (T, groups, 1), generator=g)]
    return torch.where(order < there, x, -torch.inf).view(T, E)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("shift", [-40.0, -3.0, -0.4, 0.0, 0.7, 25.0])
@pytest.mark.parametrize("E,groups", [(64, 8), (64, 32), (60, 30), (128, 8), (256, 8), (256, 32), (512, 4), (1024, 16), (96, 8)])
def test_groups_of_one_available_expert(E, groups, shift, scoring, dt):
    T, k, top = 100, 4, max(2, groups // 4)
    x = masked(T, E, groups, E + groups).to(TORCH_DT[dt])
    bias = torch.randn(E, generator=torch.Generator().manual_seed(3)) * 0.3 + shift
    k = min(k, top * (E // groups))
    want, weights, _ = route(x.double().numpy(), k, groups, top, scoring, bias.double().numpy(), 2, True, 2.5)
    idx, w = moe_router_grouped(x.cuda(), k, groups, top, scoring=scoring, bias=bias.cuda(), group_top=2, scale=2.5)
    np.testing.assert_array_equal(idx.cpu().numpy(), want)
    # exp and quotients of a few steps, softmax's sum of E terms: as in test_route_grouped_gpu.py
    np.testing.assert_allclose(w.cpu().numpy(), weights, rtol=2 * (24 + E / 32) * 2.0 ** -24, atol=1e-37)
    host = moe_router_grouped(x, k, groups, top, scoring=scoring, bias=bias, group_top=2, scale=2.5)[0]
    np.testing.assert_array_equal(host.numpy(), want)


def test_two_experts_against_one():
    """Sums 0.881 of one expert and 0.803 of two, beside a bias of -1 elsewhere: the one wins."""
    x = torch.full((1, 64), -6.0)
    x[0, :16] = -torch.inf
    x[0, 0], x[0, 8], x[0, 9] = 2.0, -0.4, -0.4
    bias = torch.zeros(64)
    bias[63] = -1.0
    assert moe_router_grouped(x.cuda(), 1, 8, 1, bias=bias.cuda())[0].item() == 0


def test_sums_a_hair_apart():
    """One expert's score against two experts' sum, apart by less than floats can tell: 64 bits decide."""
    T, E = 256, 64
    g = torch.Generator().manual_seed(1)
    x = torch.full((T, E), -torch.inf)
    x[:, 0] = torch.rand(T, generator=g) * 0.5          # sigmoid above 1/2
    bias = torch.zeros(E)
    bias[9] = -0.25
    rest = torch.sigmoid(x[:, 0].double()) + 0.25       # what experts 8 and 9 have to make: the halves of it
    x[:, 8:10] = torch.logit(rest / 2).float()[:, None]
    x[:, 0] += torch.randint(-2, 3, (T,), generator=g) * 6e-8
    want, _, _ = route(x.double().numpy(), 1, 8, 1, "sigmoid", bias.double().numpy(), 2)
    assert 20 < (want == 0).sum() < T - 20
    idx, _ = moe_router_grouped(x.cuda(), 1, 8, 1, bias=bias.cuda())
    np.testing.assert_array_equal(idx.cpu().numpy(), want)
