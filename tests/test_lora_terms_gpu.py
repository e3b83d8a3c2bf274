"""Products of numbers whose last bits are all set: what the terms of two splits leave away stays below the stated 2^-16."""
import numpy as np
import pytest
import torch

import mlx_kquant_b200 as kq
from lora_plain import check, plain
from test_lora_gpu import made

pytestmark = pytest.mark.gpu

ONES = 2.0 ** -7 - 2.0 ** -15   # behind the eight bits of a bf16 number from 1 to 2: the largest rest of sixteen bits


@pytest.mark.parametrize("T", [3, 1500])
def test_sums_next_to_the_middle_of_two_fp16_numbers(T):
    """u and b are 1 + ONES; y moves the sum over a few steps of fp16, 2^-17 at a time, so that some lie just past a middle: there an
    error of the product shows at once."""
    N = 512
    x = torch.zeros(T, 8, dtype=torch.float16, device="cuda")
    x[:, 0] = 1
    a, b = torch.zeros(1, 1, 8, device="cuda"), torch.full((1, N, 1), 1 + ONES, device="cuda")
    a[0, 0, 0] = 1 + ONES
    y = (-(2.0 ** -6) + torch.arange(N, device="cuda") * 2.0 ** -17).half().expand(T, N).contiguous()
    assert len(set(y[0].tolist())) == N
    want = plain(y, x, a, b, np.zeros(T, int), [1.0])
    check(kq.lora_update(y, x, a, b), want["y"], "y")


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_products_do_not_lean(dt):
    """Sums of positive products, over many outputs: their errors have no direction, where numbers that are cut off would all err to
    one side (by some 2^-17)."""
    T, K, N, r = 256, 256, 256, 32
    _, x, a, b, _, _ = made(3, T, K, N, r, 1, dt, "f32")
    a, b, x = a.abs(), b.abs(), x.abs()
    dy = torch.ones(T, N, dtype=x.dtype, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    out = kq.lora_update(torch.zeros_like(dy), *leaves)
    want = plain(torch.zeros_like(dy), x, a, b, np.zeros(T, int), [1.0], dy=dy)
    got = torch.autograd.grad(out, leaves, dy)
    # all rows of dy are the same, and so are those of dx: K different outputs, T N of y
    for name, g, outputs in (("y", out, T * N), ("dx", got[0], K)):
        value = want[name][0]
        lean = (g.detach().double().cpu().numpy() - value).sum() / value.sum()
        # roundings to 16 bits: half a step at most, without direction; four deviations of their mean
        rounding = 4 * {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dt] / 3 ** 0.5 / outputs ** 0.5
        assert abs(lean) < rounding + 2.0 ** -22, (name, lean)
