"""Adapters whose ranks differ in size: components of x . a^T far below a row's largest, with parameters in b as far above."""
import numpy as np
import pytest
import torch

import mlx_kquant_b200 as kq
from lora_plain import check, group_list, plain
from test_lora_gpu import TYPES, made

pytestmark = pytest.mark.gpu


def check_in_range(got, want, name):
    """check() where the value is one that the type has. fp16 ends at 65504, and 65520 rounds to infinity: a gradient of sums of 750
    entries, 1024 times as large as usual, passes that, and the nearest there is infinity with its sign."""
    value, bound = want
    beyond = np.abs(value) + bound >= (65520.0 if got.dtype == torch.float16 else np.inf)
    v = got.detach().double().cpu().numpy().reshape(value.shape)
    assert (np.sign(v[beyond]) == np.sign(value[beyond])).all() and (np.abs(v[beyond]) >= 65000).all(), name
    check(torch.where(torch.from_numpy(beyond).to(got.device).view(got.shape), 0, got), (np.where(beyond, 0.0, value), bound), name)


@pytest.mark.parametrize("T,K,N,r", [(5, 256, 64, 16), (40, 512, 72, 32), (1500, 64, 40, 8), (9, 136, 33, 100)])
@pytest.mark.parametrize("dt,pt", TYPES)
def test_components_of_many_sizes(T, K, N, r, dt, pt):
    """Powers of two from 2^-10 to 2^10 over the ranks: u's components differ a million times, their shares in y not at all."""
    y, x, a, b, s, dy = made(T + r, T, K, N, r, 2, dt, pt)
    ids = torch.arange(T, dtype=torch.int32, device="cuda") % 2
    size = torch.exp2(torch.linspace(-10, 10, r).round()).cuda()
    for up in (True, False):
        f = size if up else 1 / size
        a2, b2 = (a.float() * f[:, None]).to(a.dtype), (b.float() / f).to(b.dtype)
        want = plain(y, x, a2, b2, group_list(ids.cpu().numpy(), 1, None, 2, 1, T), s.cpu().numpy(), dy=dy)
        leaves = [t.clone().requires_grad_() for t in (x, a2, b2)]
        out = kq.lora_update(y, *leaves, ids, s)
        check(out, want["y"], "y")
        check(kq.lora_update(y, x, a2, b2, ids, s), want["y"], "y without gradients")
        for name, g in zip(("dx", "da", "db"), torch.autograd.grad(out, leaves, dy)):
            check_in_range(g, want[name], name)


@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -100, 2.0 ** 60, 2.0 ** 100])
def test_factors_far_from_one(size):
    """v beyond the range of fp16 by a factor that the matrices take back."""
    T, K, N, r = 9, 128, 64, 8
    y, x, a, b, s, dy = made(1, T, K, N, r, 1, "f16", "f32")
    a = a * size
    want = plain(y, x, a, b / size, np.zeros(T, int), s.cpu().numpy(), dy=dy)
    leaves = [t.clone().requires_grad_() for t in (x, a, b / size)]
    out = kq.lora_update(y, *leaves, None, s)
    check(out, want["y"], "y")
    for name, g in zip(("dx", "da", "db"), torch.autograd.grad(out, leaves, dy)):
        check(g, want[name], name)
