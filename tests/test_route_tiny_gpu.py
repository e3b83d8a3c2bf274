"""Gradient of softmax scores that are renormalised over next to nothing: the sum's 1e-20 counts, and experts not picked have a share."""
import numpy as np
import pytest
import torch

from gpu_util import TORCH_DT
from mlx_kquant_b200.moe import moe_router_grouped
from route_plain import route


def whole_gradient(scores, idx, dw, scale):
    """d sum(w dw) / dl of w_j = scale s_ij / (S + 1e-20), softmax, all of it: s_e ([e picked] ds_e - sum_j ds_j s_ij)."""
    dl = np.zeros_like(scores)
    for t in range(scores.shape[0]):
        s, d = scores[t][idx[t]], scale * dw[t]
        S = s.sum() + 1e-20
        ds = (d - (d * s / S).sum()) / S
        dl[t] = -scores[t] * (ds * s).sum()
        dl[t, idx[t]] += ds * s
    return dl


def made(low, T=40, E=32, k=4, seed=0):
    """Four experts with nearly all of the softmax and a bias that keeps them from being picked, the others `low` below."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, E, generator=g) * 0.5 - low
    x[:, :4] = torch.randn(T, 4, generator=g) * 0.5 - 2.0
    x[:, 0] = 0.0                                        # the largest: differences from it are exact
    bias = torch.zeros(E)
    bias[:4] = -2.0
    return x, bias, torch.randn(T, k, generator=g)


def test_the_formula_has_the_gradient_of_its_weights():
    """Central differences of the 64-bit weights, picks held."""
    x, bias, dw = (t.double().numpy() for t in made(45.5, T=4))
    idx, _, scores = route(x, 4, scoring="softmax", bias=bias, scale=1.5)
    dl = whole_gradient(scores, idx, dw, 1.5)
    for t in range(4):
        for e in range(32):
            side = []
            for h in (1e-5, -1e-5):
                y = x.copy()
                y[t, e] += h
                p = np.exp(y[t] - y[t].max())
                p = (p / p.sum())[idx[t]]
                side.append((1.5 * p / (p.sum() + 1e-20) * dw[t]).sum())
            # the difference's third-order term h^2 / 6 and the weights' rounding 2^-53 / h
            assert abs((side[0] - side[1]) / 2e-5 - dl[t, e]) < 1e-9


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("low", [5.0, 25.0, 28.5, 35.0, 45.5, 50.0, 70.0])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_scores_next_to_nothing(device, low, dt):
    x, bias, dw = made(low)
    x = x.to(TORCH_DT[dt])
    idx, w, scores = route(x.double().numpy(), 4, scoring="softmax", bias=bias.double().numpy(), scale=1.5)
    want = whole_gradient(scores, idx, dw.double().numpy(), 1.5)
    leaf = x.to(device).requires_grad_()
    gi, gw = moe_router_grouped(leaf, 4, scoring="softmax", bias=bias.to(device), scale=1.5)
    np.testing.assert_array_equal(gi.cpu().numpy(), idx)
    dl, = torch.autograd.grad(gw, leaf, dw.to(device))
    got = dl.double().cpu().numpy()
    # float32: 25 steps of 2^-24 for a score, four of them in a product of scores, times the parts that are subtracted; of the share of
    # experts not picked, half a step of the row's mean may be left away
    half = 2.0 ** -24 if dt == "f32" else 2.0 ** -8
    for t in range(x.shape[0]):
        s = scores[t][idx[t]]
        S, d = s.sum() + 1e-20, 1.5 * np.abs(dw[t].double().numpy())
        mean = (d * s / S).sum()
        parts = scores[t] * mean * 1e-20 / S
        parts[idx[t]] += s / S * (d + mean)
        if device == "cpu":      # torch subtracts sum_j ds_j s_j as it comes: what is left of sizes ds_j s_j has their rounding, times s_e
            parts = parts + scores[t] * (s / S * (d + mean)).sum()
        off = np.abs(got[t] - want[t])
        assert (off <= half * np.abs(want[t]) + 100 * 2.0 ** -24 * parts + 2.0 ** -24 * mean + 1e-37).all(), (t, off.max())
    if dt == "f32" and low == 45.5:
        assert np.abs(want[:, 0]).max() > 0.1            # the largest expert, not picked, has a full share
