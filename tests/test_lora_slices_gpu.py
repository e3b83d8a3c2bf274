"""Gradients of rows that a token's slots share, so many that dx is made a few columns at a time."""
import numpy as np
import pytest
import torch

from lora_plain import check, group_list, plain
from mlx_kquant_b200 import _lib
from mlx_kquant_b200.moe import gather_lora_update
from test_lora_gpu import TYPES, made

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K,N", [(1000, 40), (1000, 41), (1001, 40)])
@pytest.mark.parametrize("dt,pt", TYPES)
def test_columns_in_turns(K, N, dt, pt):
    T, R, E, G, r = 4125, 8, 6, 2, 12
    y, x, a, b, s, dy = made(7, T, K, N, r, G, dt, pt, E, R)
    rng = np.random.default_rng(3)
    experts, ids = rng.integers(-1, E + 1, (T, R)).astype(np.int32), rng.integers(-1, G, T).astype(np.int32)
    # fewer columns at once than there are, by the workspace: three turns, the last one short
    pcode = _lib.KQ_F32 if pt == "f32" else _lib.KQ_F16
    shared = _lib.lib().kq_lora_backward_workspace_bytes(T * R, R, 1, K, N, r, pcode) - _lib.lib().kq_lora_backward_workspace_bytes(T * R, 1, 0, K, N, r, pcode)
    assert shared == T * R * 448 * 4
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    out = gather_lora_update(y, *leaves, torch.from_numpy(experts).cuda(), torch.from_numpy(ids).cuda(), s)
    dx, da, db = torch.autograd.grad(out, leaves, dy)
    some = np.unique(np.concatenate([[0, 1, 2, T - 2, T - 1], rng.integers(0, T, 60)]))
    at = torch.from_numpy(some).cuda()
    n = len(some)
    want = plain(y[at].reshape(n * R, N), x[at], a.reshape(G * E, r, K), b.reshape(G * E, N, r), group_list(ids[some], R, experts[some], G, E, n),
                 np.repeat(s.cpu().numpy(), E), R, True, dy[at].reshape(n * R, N))
    check(out[at], want["y"], "y")
    check(dx[at], want["dx"], "dx")
    assert not dx[torch.from_numpy(ids < 0).cuda()].any()
    # all of the matrices' gradients, in 64 bits on the GPU: sums of up to some 5000 entries, as lora_plain.py bounds them in the norm
    group = torch.from_numpy(group_list(ids, R, experts, G, E, T)).cuda()
    xd, ad, bd, dyd = x.double(), a.double().view(-1, r, K), b.double().view(-1, N, r), dy.double().view(-1, N)
    da_want, db_want = torch.zeros_like(ad), torch.zeros_like(bd)
    for g in range(G * E):
        e = torch.nonzero(group == g)[:, 0]
        rows, f = xd[e // R], s[g // E].double()
        da_want[g], db_want[g] = f * (dyd[e] @ bd[g]).T @ rows, f * dyd[e].T @ (rows @ ad[g].T)
    for got, exact in ((da, da_want), (db, db_want)):
        most = {torch.float32: 4e-6, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[got.dtype]
        assert (got.double().view(exact.shape) - exact).norm() <= most * exact.norm()
