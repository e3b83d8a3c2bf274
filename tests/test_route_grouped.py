"""moe_router_grouped on host tensors against the 64-bit statement (route_plain.py), and its refusals."""
import numpy as np
import pytest
import torch

from mlx_kquant_b200 import _lib
from mlx_kquant_b200.moe import moe_router_grouped
from route_plain import gradient, route

CASES = [(5, 16, 4, 4, 2, "sigmoid", True, 2, True), (3, 12, 3, 4, 3, "softmax", False, 1, False), (4, 8, 8, 1, 1, "softmax", True, 2, True),
         (6, 10, 2, 5, 1, "sigmoid", False, 2, False), (2, 1, 1, 1, 1, "sigmoid", False, 1, True)]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_host_tensors(case):
    T, E, k, groups, top, scoring, biased, group_top, norm = case
    g = torch.Generator().manual_seed(E)
    x = torch.randn(T, E, generator=g)
    x[0, :E // 2] = float("-inf")
    x[T - 1] = float("-inf")
    bias = torch.randn(E, generator=g) * 0.2 if biased else None
    want, w, scores = route(x.double().numpy(), k, groups, top, scoring, None if bias is None else bias.double().numpy(), group_top, norm, 1.5)
    leaf = x.clone().requires_grad_()
    idx, got = moe_router_grouped(leaf, k, groups, top, scoring=scoring, bias=bias, group_top=group_top, norm_topk_prob=norm, scale=1.5)
    assert idx.dtype == torch.int32 and np.array_equal(idx.numpy(), want)
    np.testing.assert_allclose(got.detach().numpy(), w, rtol=2e-6, atol=1e-30)
    rows = slice(1, T - 1)                         # rows without -inf: torch has no gradient at the others
    dw = torch.randn(T, k, generator=g)
    leaf = x[rows].clone().requires_grad_()
    _, got = moe_router_grouped(leaf, k, groups, top, scoring=scoring, bias=bias, group_top=group_top, norm_topk_prob=norm, scale=1.5)
    dl, = torch.autograd.grad(got, leaf, dw[rows])
    np.testing.assert_allclose(dl.numpy(), gradient(x[rows].double().numpy(), want[rows], dw[rows].double().numpy(), scoring, norm, 1.5, scores[rows]),
                               rtol=1e-4, atol=1e-6)


def test_the_statement_has_the_gradient_of_its_weights():
    """The formula against central differences of the weights, picks held: 64 bits, a step of 1e-6."""
    rng = np.random.default_rng(1)
    x, dw = rng.normal(0, 1, (3, 9)), rng.normal(0, 1, (3, 4))
    for scoring in ("sigmoid", "softmax"):
        for norm in (True, False):
            idx, _, scores = route(x, 4, scoring=scoring, norm=norm, scale=2.0)
            dl = gradient(x, idx, dw, scoring, norm, 2.0, scores)
            for t in range(3):
                for e in range(9):
                    side = []
                    for h in (1e-6, -1e-6):
                        y = x.copy()
                        y[t, e] += h
                        moved, w, _ = route(y, 4, scoring=scoring, norm=norm, scale=2.0)
                        assert np.array_equal(moved, idx)
                        side.append((w * dw).sum())
                    assert abs((side[0] - side[1]) / 2e-6 - dl[t, e]) < 1e-7


def test_refusals():
    x = torch.zeros(2, 12)
    for args, kw, words in (((x, 2), dict(scoring="tanh"), "scoring"), ((x, 13), {}, "top_k"), ((x, 0), {}, "top_k"),
                            ((torch.zeros(2, 64), 33), {}, "top_k"), ((torch.zeros(2, 1025), 2), {}, "1024"),
                            ((x, 2, 5, 1), {}, "multiple"), ((x, 2, 4, 5), {}, "top_groups"), ((x, 2, 4, 0), {}, "top_groups"),
                            ((x, 4, 4, 1), {}, "fewer"), ((x, 2), dict(group_top=3), "group_top"), ((x[0], 2), {}, "T, E"),
                            ((x.int(), 2), {}, "floating"), ((x, 2), dict(bias=torch.zeros(11)), "bias")):
        with pytest.raises(ValueError, match=words):
            moe_router_grouped(*args, **kw)
    L, bad, p = _lib.lib(), _lib.KQ_ERR_INVALID_ARGUMENT, 256   # never followed
    call = lambda E=12, k=2, G=1, top=1, gt=2, sc=b"sigmoid", dt=0, T=2, logits=p: L.kq_moe_router_grouped(  # noqa: E731
        logits, dt, T, E, k, G, top, gt, sc, None, 1, 1.0, p, p, None)
    for kw in (dict(E=0), dict(E=1025), dict(k=0), dict(k=13), dict(E=64, k=33), dict(G=5), dict(G=0), dict(G=4, top=5), dict(G=4, top=0),
               dict(G=6, top=1, k=3), dict(gt=0), dict(gt=3), dict(sc=b"tanh"), dict(dt=3), dict(T=-1), dict(T=2 ** 31), dict(logits=None)):
        assert call(**kw) == bad, kw
        assert b"[mlx_kquant.moe_router_grouped]" in L.kq_last_error()
    assert call(T=0) == 0
    assert L.kq_moe_router_grouped_backward(None, 0, 2, 12, 2, b"softmax", 1, 1.0, p, p, p, None) == bad
