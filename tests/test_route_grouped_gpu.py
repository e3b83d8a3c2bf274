"""moe_router_grouped on the GPU: the same picks as 64 bits make, weights and gradients of the formulas."""
import numpy as np
import pytest
import torch

from gpu_util import TORCH_DT
from mlx_kquant_b200.moe import moe_glu, moe_router_grouped, route_topk
from route_plain import gradient, route

pytestmark = pytest.mark.gpu

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# T, E, top_k, groups, top_groups, scoring, bias, group_top, norm
CASES = [(1, 256, 8, 8, 4, "sigmoid", True, 2, True), (61, 160, 6, 8, 3, "softmax", False, 1, False), (33, 128, 8, 1, 1, "softmax", False, 1, True),
         (17, 1, 1, 1, 1, "sigmoid", True, 2, True), (9, 7, 3, 1, 1, "softmax", True, 1, False), (40, 60, 4, 4, 2, "sigmoid", False, 2, False),
         (5, 1024, 32, 16, 5, "sigmoid", True, 2, True), (6, 1000, 12, 40, 3, "softmax", True, 2, True), (300, 64, 2, 64, 7, "sigmoid", True, 2, True),
         (12, 384, 8, 3, 1, "softmax", False, 2, True), (129, 33, 32, 1, 1, "sigmoid", False, 1, True), (4, 512, 10, 2, 2, "softmax", False, 1, True)]


def run(x, case, bias, dw=None, scale=2.5):
    T, E, k, groups, top, scoring, _, group_top, norm = case
    leaf = x.detach().requires_grad_() if dw is not None else x
    idx, w = moe_router_grouped(leaf, k, groups, top, scoring=scoring, bias=bias, group_top=group_top, norm_topk_prob=norm, scale=scale)
    return (idx, w) if dw is None else (idx, w.detach(), torch.autograd.grad(w, leaf, dw)[0])


def against_plain(x, case, bias, dt, dw):
    """float32 scores: exp and the quotients are off by a few steps, sums by one a term of a tree - 16 steps of 2^-24 in all, E / 32 + 5
    more of softmax's sum; a gradient is a difference of such numbers, so its bound goes by the sizes of what is subtracted."""
    T, E, k, groups, top, scoring, _, group_top, norm = case
    xd = x.detach().double().cpu().numpy()
    want, w, scores = route(xd, k, groups, top, scoring, None if bias is None else bias.double().cpu().numpy(), group_top, norm, 2.5)
    idx, got, dl = run(x, case, bias, dw)
    assert idx.dtype == torch.int32 and got.dtype == torch.float32 and dl.dtype == x.dtype
    np.testing.assert_array_equal(idx.cpu().numpy(), want)
    steps = (24 + E / 32) * 2.0 ** -24
    np.testing.assert_allclose(got.cpu().numpy(), w, rtol=steps * 2, atol=1e-37)
    d = dw.double().cpu().numpy()
    exact = gradient(xd, want, d, scoring, norm, 2.5, scores)
    size = gradient(xd, want, np.abs(d), scoring, False, 2.5, scores)      # without the difference: how large its parts are
    parts = np.abs(size)
    if norm:
        S = np.array([scores[t][want[t][want[t] >= 0]].sum() + 1e-20 for t in range(T)])
        parts = np.zeros_like(exact)
        for t in range(T):
            on = want[t][want[t] >= 0]
            parts[t, on] = 2.5 * np.abs(d[t]).max() * 2 * scores[t][on] / S[t]
    elif scoring == "softmax":
        for t in range(T):
            on = want[t] >= 0
            parts[t] = scores[t] * 2.5 * (np.abs(d[t][on]) * scores[t][want[t][on]]).sum()
            parts[t, want[t][on]] += 2.5 * np.abs(d[t][on]) * scores[t][want[t][on]]
    off = np.abs(dl.double().cpu().numpy() - exact)
    tiny = {"f32": 1e-37, "f16": 2.0 ** -25, "bf16": 1e-37}[dt]
    assert (off <= HALF[dt] * np.abs(exact) + 4 * steps * parts + tiny).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_picks_weights_gradient(case, dt):
    T, E, k = case[:3]
    g = torch.Generator().manual_seed(T + E)
    x = (torch.randn(T, E, generator=g) * 1.5).to(TORCH_DT[dt]).cuda()
    bias = (torch.randn(E, generator=g) * 0.1).cuda() if case[6] else None
    dw = torch.randn(T, k, generator=g).cuda()
    against_plain(x, case, bias, dt, dw)
    # many experts alike: the lowest index first; with a bias of few values the sums are alike too
    x = (torch.randint(-2, 3, (T, E), generator=g) * 0.5).to(TORCH_DT[dt]).cuda()
    bias = (torch.randint(0, 3, (E,), generator=g) * 0.25).cuda() if case[6] else None
    against_plain(x, case, bias, dt, dw)
    # experts that are not available, of some rows all, some with the type's lowest value
    x = (torch.randn(T, E, generator=g) * 1.5).to(TORCH_DT[dt])
    x[torch.rand(T, E, generator=g) < 0.7] = float("-inf")
    x[T // 2] = float("-inf")
    x[torch.rand(T, E, generator=g) < 0.1] = torch.finfo(TORCH_DT[dt]).min
    against_plain(x.cuda(), case, bias, dt, dw)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_scores_that_floats_cannot_tell_apart(scoring):
    """Score + bias whose order hangs on bits below float32's last: 64 bits decide, ties still go by the index."""
    T, E, k = 400, 256, 8
    g = torch.Generator().manual_seed(3)
    base = torch.randn(T, 1, generator=g)
    x = base + torch.randint(0, 3, (T, E), generator=g) * 1e-7   # neighbouring floats
    bias = torch.ones(E)
    case = (T, E, k, 8, 4, scoring, True, 2, True)
    against_plain(x.cuda(), case, bias.cuda(), "f32", torch.randn(T, k, generator=g).cuda())
    bias = 1 + torch.randint(0, 2, (E,), generator=g) * 2.0 ** -23
    against_plain(x.cuda(), case, bias.cuda(), "f32", torch.randn(T, k, generator=g).cuda())


def test_nan_and_infinity():
    x = torch.randn(4, 64).cuda()
    x[1, 40] = float("nan")
    x[2, 9] = float("inf")
    for scoring in ("sigmoid", "softmax"):
        for bias in (None, torch.zeros(64).cuda()):
            idx, w = moe_router_grouped(x, 4, 8, 3, scoring=scoring, bias=bias)
            ref, wr = moe_router_grouped(torch.cat([x[:1], x[3:]]), 4, 8, 3, scoring=scoring, bias=bias)
            assert torch.equal(idx[[0, 3]], ref) and torch.equal(w[[0, 3]], wr)
            assert torch.isnan(w[1]).all()
            assert ((idx >= 0) & (idx < 64)).all() and all(len(set(r)) == 4 for r in idx.tolist())
            if scoring == "sigmoid":
                assert idx[1, 0] == 40 and idx[2, 0] == 9 and torch.isfinite(w[2]).all()


def test_views_streams_and_a_graph():
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn(50, 300, device="cuda", generator=g)
    x = wide[:, 7:263]
    bias = torch.randn(256, device="cuda", generator=g) * 0.1
    dw = torch.randn(50, 8, device="cuda", generator=g)
    case = (50, 256, 8, 8, 4, "sigmoid", True, 2, True)
    first = run(x.contiguous(), case, bias, dw)
    for p, q in zip(first, run(x, case, bias.double(), dw)):
        assert torch.equal(p, q)
    assert torch.equal(first[0], run(x.to(torch.float32), case, bias)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(x, case, bias, dw)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(first, again):
        assert torch.equal(p, q)
    leaf = x.contiguous().requires_grad_()
    moe_router_grouped(leaf, 8, 8, 4, bias=bias)   # an eager graph of the leaf, gone again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        idx, w = moe_router_grouped(leaf, 8, 8, 4, bias=bias)
        dl, = torch.autograd.grad(w, leaf, dw)
    with torch.no_grad():
        leaf.copy_(leaf.flip(0))
    graph.replay()
    idx2, w2, dl2 = run(leaf, case, bias, dw, 1.0)
    assert torch.equal(idx, idx2) and torch.equal(w, w2) and torch.equal(dl, dl2)
    # picks alone, or an empty batch
    assert torch.autograd.grad(moe_router_grouped(leaf, 8, 8, 4)[1].sum(), leaf)[0].shape == leaf.shape
    e_idx, e_w = moe_router_grouped(leaf[:0], 8, 8, 4, bias=bias)
    assert e_idx.shape == e_w.shape == (0, 8)


def test_same_routing_as_the_plain_router():
    x = torch.randn(200, 128, device="cuda")
    idx, w = moe_router_grouped(x, 8, scoring="softmax")
    ref, wr = route_topk(x, 8)
    assert torch.equal(idx, ref)
    torch.testing.assert_close(w, wr, rtol=1e-5, atol=0)


def test_host_and_device_agree():
    g = torch.Generator().manual_seed(9)
    x, bias = torch.randn(64, 96, generator=g), torch.randn(96, generator=g) * 0.1
    x[3, :] = float("-inf")
    x[4, 5:] = float("-inf")
    for scoring in ("sigmoid", "softmax"):
        for group_top in (1, 2):
            h = moe_router_grouped(x, 6, 8, 3, scoring=scoring, bias=bias, group_top=group_top)
            d = moe_router_grouped(x.cuda(), 6, 8, 3, scoring=scoring, bias=bias, group_top=group_top)
            assert torch.equal(h[0], d[0].cpu())
            torch.testing.assert_close(h[1], d[1].cpu(), rtol=1e-5, atol=1e-37)


@pytest.mark.parametrize("T", [3, 200])
def test_rows_that_run_out_of_experts_reach_the_block(T):
    """Index -1 with weight 0 in the fused block, small and large: as if the row had fewer experts."""
    from gpu_util import mint_wire
    rng = np.random.default_rng(2)
    E, H, F, k = 8, 256, 256, 4
    mk = lambda n, d: torch.from_numpy(np.stack([mint_wire("q4_k", rng.normal(0, d ** -0.5, (n, d)).astype(np.float32)) for _ in range(E)])).cuda()  # noqa: E731
    wg, wu, wd = mk(F, H), mk(F, H), mk(H, F)
    x = torch.from_numpy(rng.normal(0, 1, (T, H)).astype(np.float32)).bfloat16().cuda()
    logits = torch.from_numpy(rng.normal(0, 1, (T, E)).astype(np.float32))
    logits[0] = float("-inf")
    logits[1, 2:] = float("-inf")
    idx, w = moe_router_grouped(logits.cuda(), k)
    y = moe_glu(x, wg, wu, wd, "q4_k", idx, w)
    assert (y[0] == 0).all() and torch.isfinite(y).all()
    full = torch.where(idx < 0, 0, idx)            # weight 0 on some other expert
    torch.testing.assert_close(y.float(), moe_glu(x, wg, wu, wd, "q4_k", full, w).float(), rtol=0.02, atol=0.01)


@pytest.mark.parametrize("group_top", [1, 2])
def test_many_doubtful_tokens(group_top):
    """Logits and biases of few values a hair apart, so that most tokens are ranked again, some with more than 32 experts in doubt."""
    g = torch.Generator().manual_seed(group_top)
    T, E, k = 700, 256, 8
    for step, few in ((2.0 ** -22, 4), (2.0 ** -23, 2), (2.0 ** -18, 40)):
        x = 0.75 + torch.randint(0, few, (T, E), generator=g) * step
        x[::3] += torch.randn(x[::3].shape, generator=g)
        bias = 0.125 + torch.randint(0, few, (E,), generator=g) * step * 0.5
        case = (T, E, k, 8, 4, "sigmoid", True, group_top, True)
        xd = x.double().numpy()
        want, _, _ = route(xd, k, 8, 4, "sigmoid", bias.double().numpy(), group_top)
        np.testing.assert_array_equal(run(x.cuda(), case, bias.cuda())[0].cpu().numpy(), want)
        want, _, _ = route(xd, k, 8, 4, "sigmoid", None, group_top)
        np.testing.assert_array_equal(run(x.cuda(), case, None)[0].cpu().numpy(), want)
