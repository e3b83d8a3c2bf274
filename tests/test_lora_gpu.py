"""Low-rank adapters against the 64-bit statement (lora_plain.py): sizes, types, masks, strides, gradients, streams, graphs."""
import numpy as np
import pytest
import torch

import mlx_kquant_b200 as kq
from gpu_util import TORCH_DT
from lora_plain import check, group_list, plain
from mlx_kquant_b200.moe import gather_lora_update

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")]


def made(seed, T, K, N, r, G, dt, pt, E=None, slots=None, shared=True):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = rnd(T, K) if slots is None or shared else rnd(T, slots, K)
    y = rnd(T, N) if slots is None else rnd(T, slots, N)
    lead = (G,) if E is None else (G, E)
    a, b = rnd(*lead, r, K) * K ** -0.5, rnd(*lead, N, r) * 0.1
    s = torch.rand(G, generator=g) + 0.5
    dy = rnd(*y.shape)
    dt, pt = TORCH_DT[dt], TORCH_DT[pt]
    return [t.cuda() for t in (y.to(dt), x.to(dt), a.to(pt), b.to(pt), s, dy.to(dt))]


def some_ids(seed, T, G):
    """adapters in no order, some rows without one, in all the ways to say so"""
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, G, T)
    out = rng.random(T) < 0.2
    return np.where(out, rng.choice([-1, G, -7, 2 ** 31 - 1], T), ids).astype(np.int32)


SIZES = [(1, 256, 256, 16, 1), (1, 4096, 512, 16, 3), (2, 32, 8, 1, 2), (7, 33, 17, 3, 2), (16, 64, 64, 8, 1), (17, 264, 1000, 12, 5),
         (61, 512, 1432, 32, 32), (70, 48, 1032, 100, 2), (129, 72, 100, 5, 3), (200, 100, 129, 33, 2), (300, 1024, 96, 64, 7),
         (513, 136, 72, 128, 3), (1000, 96, 264, 24, 1), (2100, 64, 40, 16, 40)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dt,pt", TYPES)
def test_update_and_gradients(size, dt, pt):
    T, K, N, r, G = size
    y, x, a, b, s, dy = made(sum(size), T, K, N, r, G, dt, pt)
    ids = some_ids(T, T, G) if G > 1 else None
    dev_ids = None if ids is None else torch.from_numpy(ids).cuda()
    want = plain(y, x, a, b, group_list(ids, 1, None, G, 1, T), s.cpu().numpy(), dy=dy)
    check(kq.lora_update(y, x, a, b, dev_ids, s), want["y"], "y")
    leaves = [t.clone().requires_grad_() for t in (y, x, a, b)]
    out = kq.lora_update(*leaves, dev_ids, s)
    check(out, want["y"], "y beside gradients")
    gy, dx, da, db = torch.autograd.grad(out, leaves, dy)
    assert torch.equal(gy, dy)
    for name, got in (("dx", dx), ("da", da), ("db", db)):
        assert got.shape == leaves[1 + ("dx", "da", "db").index(name)].shape
        check(got, want[name], name)


EXPERT_SIZES = [(1, 1, 1, 64, 64, 4, 1), (1, 8, 128, 256, 96, 8, 2), (5, 3, 7, 33, 21, 6, 2), (9, 8, 16, 512, 264, 16, 4),
                (40, 4, 8, 128, 72, 40, 1), (130, 6, 60, 264, 136, 8, 3), (700, 8, 32, 64, 48, 16, 1)]


@pytest.mark.parametrize("size", EXPERT_SIZES, ids=str)
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("dt,pt", TYPES)
def test_update_beside_experts(size, shared, dt, pt):
    T, R, E, K, N, r, G = size
    y, x, a, b, s, dy = made(sum(size), T, K, N, r, G, dt, pt, E, R, shared)
    rng = np.random.default_rng(T)
    ids = some_ids(T, T, G) if G > 1 else None
    experts = rng.integers(0, E, (T, R))            # an expert may come twice in a row
    experts[rng.random((T, R)) < 0.1] = -1
    experts[rng.random((T, R)) < 0.05] = E
    idx = torch.from_numpy(experts.astype(np.int32)).cuda()
    dev_ids = None if ids is None else torch.from_numpy(ids).cuda()
    want = plain(y.reshape(T * R, N), x.reshape(-1, K), a.reshape(G * E, r, K), b.reshape(G * E, N, r), group_list(ids, R, experts, G, E, T),
                 np.repeat(s.cpu().numpy(), E), R, shared, dy.reshape(T * R, N))
    check(gather_lora_update(y, x, a, b, idx, dev_ids, s), want["y"], "y")
    leaves = [t.clone().requires_grad_() for t in (y, x, a, b)]
    out = gather_lora_update(*leaves, idx, dev_ids, s)
    check(out, want["y"], "y beside gradients")
    _, dx, da, db = torch.autograd.grad(out, leaves, dy)
    for name, got in (("dx", dx), ("da", da), ("db", db)):
        check(got, want[name], name)


@pytest.mark.parametrize("T", [5, 400])
def test_rows_without_an_adapter_keep_their_bits(T):
    y, x, a, b, s, dy = made(3, T, 64, 72, 8, 2, "bf16", "bf16")
    none = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(kq.lora_update(y, x, a, b, none, s), y)
    mixed = none.clone()
    mixed[1::3] = 1
    a[0].fill_(float("nan"))                       # nobody's adapter
    out = kq.lora_update(y, x, a, b, mixed, s)
    assert torch.equal(out[mixed < 0], y[mixed < 0]) and torch.isfinite(out).all() and not torch.equal(out, y)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    dx, da, db = torch.autograd.grad(kq.lora_update(y, *leaves, mixed, s), leaves, dy)
    assert (dx[mixed < 0] == 0).all() and (da[0] == 0).all() and (db[0] == 0).all() and torch.isfinite(dx).all()
    buf = y.clone()
    assert kq.lora_update(buf, x, a, b, mixed, s, out=buf) is buf and torch.equal(buf, out)


def test_infinities_stay_in_their_rows():
    for T in (6, 300):
        y, x, a, b, s, _ = made(4, T, 64, 72, 8, 2, "f16", "f16")
        ids = torch.arange(T, device="cuda", dtype=torch.int32) % 2
        clean = kq.lora_update(y, x, a, b, ids, s)
        x[3, 5], x[1, 7], y[2, 4] = float("inf"), float("nan"), float("-inf")
        out = kq.lora_update(y, x, a, b, ids, s)
        keep = [t for t in range(T) if t not in (1, 2, 3)]
        assert torch.equal(out[keep], clean[keep])
        assert torch.isnan(out[1]).all() and not torch.isfinite(out[3]).any()
        assert out[2, 4] == float("-inf") and torch.equal(out[2, 5:], clean[2, 5:])


def test_large_values_and_small_ones_in_fp16():
    """u beyond the range of fp16 beside outputs inside it; parameters that fp16 holds with few bits."""
    y, x, a, b, s, _ = made(5, 9, 512, 64, 16, 1, "f16", "f16")
    x, a, b = x * 16, a * 512, b * 2.0 ** -14      # u of some 1e5
    want = plain(y, x, a, b, np.zeros(9, int), s.cpu().numpy())
    check(kq.lora_update(y, x, a, b, None, s), want["y"])
    y, x, a, b, s, _ = made(6, 9, 512, 64, 16, 1, "f16", "f32")
    a = a * 1e-6
    b = b * 1e6
    check(kq.lora_update(y, x, a, b, None, s), plain(y, x, a, b, np.zeros(9, int), s.cpu().numpy())["y"])


def test_strides_and_shapes():
    dt = torch.bfloat16
    y, x, a, b, s, dy = made(7, 24, 64, 40, 8, 3, "bf16", "bf16")
    ids = torch.arange(24, device="cuda", dtype=torch.int32) % 3
    want = kq.lora_update(y, x, a, b, ids, s)
    wide = torch.zeros(24, 131, dtype=dt, device="cuda")
    for lo in (0, 1, 8, 64):                       # rows that start anywhere, odd strides
        wide[:, lo:lo + 64] = x
        assert torch.equal(kq.lora_update(y, wide[:, lo:lo + 64], a, b, ids, s), want)
        wy = torch.zeros(24, 107, dtype=dt, device="cuda")
        wy[:, lo:lo + 40] = y
        assert torch.equal(kq.lora_update(wy[:, lo:lo + 40], x, a, b, ids, s), want)
    assert torch.equal(kq.lora_update(y.T.contiguous().T, x.T.contiguous().T, a, b, ids, s), want)
    assert torch.equal(kq.lora_update(y, x, a.transpose(1, 2).contiguous().transpose(1, 2), b, ids, s), want)
    shaped = kq.lora_update(y.view(4, 3, 2, 40), x.view(4, 3, 2, 64), a, b, ids.view(4, 3, 2), s)
    assert torch.equal(shaped.view(24, 40), want)
    per = torch.tensor([2, 0, -1, 1], device="cuda")   # one index for six rows, int64
    assert torch.equal(kq.lora_update(y.view(4, 6, 40), x.view(4, 6, 64), a, b, per, s).view(24, 40),
                       kq.lora_update(y, x, a, b, per.repeat_interleave(6), s))
    one = kq.lora_update(y[0], x[0], a[1], b[1], scaling=float(s[1]))
    assert torch.equal(one, kq.lora_update(y[:1], x[:1], a, b, torch.tensor([1], device="cuda"), s)[0])
    far = torch.full((24,), 2 ** 32, device="cuda")    # not adapter 0
    assert torch.equal(kq.lora_update(y, x, a, b, far, s), y)
    f32 = kq.lora_update(y, x.float(), a, b, ids, s)
    assert torch.equal(f32, want)
    assert kq.lora_update(y[:0], x[:0], a, b, ids[:0], s).shape == (0, 40)
    # a gradient that is one value, expanded
    leaf = a.clone().requires_grad_()
    ga, = torch.autograd.grad(kq.lora_update(y, x, leaf, b, ids, s).sum(), leaf)
    gb, = torch.autograd.grad(kq.lora_update(y, x, leaf, b, ids, s), leaf, torch.ones_like(y))
    assert torch.equal(ga, gb)


def test_refusals_on_the_gpu():
    y, x, a, b, s, _ = made(8, 4, 32, 24, 4, 2, "bf16", "bf16")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="scaling must be"):
        kq.lora_update(y, x, a, b, ids, s[:1])
    with pytest.raises(ValueError, match="no gradient"):
        kq.lora_update(y, x, a, b, ids, s.clone().requires_grad_())
    with pytest.raises(ValueError, match="out must be"):
        kq.lora_update(y, x, a, b, ids, s, out=y[:, :12])
    with pytest.raises(ValueError, match="out must be"):
        kq.lora_update(y, x, a, b, ids, s, out=torch.empty(24, 4, dtype=y.dtype, device="cuda").T)
    leaf = a.clone().requires_grad_()
    with pytest.raises(ValueError, match="out="):
        kq.lora_update(y, x, leaf, b, ids, s, out=y)
    with pytest.raises(ValueError, match="stream="):
        kq.lora_update(y, x, leaf, b, ids, s, stream=torch.cuda.Stream())
    with torch.no_grad():
        kq.lora_update(y, x, leaf, b, ids, s, out=torch.empty_like(y), stream=torch.cuda.Stream())
    torch.cuda.synchronize()


@pytest.mark.parametrize("T", [12, 700])
def test_same_bits_again_and_on_another_stream(T):
    y, x, a, b, s, dy = made(9, T, 256, 264, 16, 3, "bf16", "f32")
    ids = torch.from_numpy(some_ids(1, T, 3)).cuda()
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]

    def both():
        out = kq.lora_update(y, *leaves, ids, s)
        return (out, *torch.autograd.grad(out, leaves, dy))

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = both()
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(first, second):
        assert torch.equal(p, q)
    # an operand that the current stream has yet to make
    big = torch.randn(4096, 4096, device="cuda")
    x2 = torch.zeros_like(x)
    for _ in range(3):
        big = big @ big * 1e-3
    x2.copy_(x)
    out = kq.lora_update(y, x2, a, b, ids, s, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(out, first[0])


@pytest.mark.parametrize("T", [3, 300])
def test_captured_step(T):
    """Forward and backward in a graph, behind an eager step of the same leaves; replayed on new values of the inputs."""
    y, x, a, b, s, dy = made(10, T, 128, 136, 8, 2, "bf16", "f32")
    ids = torch.from_numpy(some_ids(2, T, 2)).cuda()
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    torch.autograd.grad(kq.lora_update(y, *leaves, ids, s), leaves, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(kq.lora_update(y, *leaves, ids, s), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kq.lora_update(y, *leaves, ids, s)
        grads = torch.autograd.grad(out, leaves, dy)
    with torch.cuda.graph(other):                  # a second one, replayed in between
        out2 = kq.lora_update(y, x, a, b, ids, s)
    with torch.no_grad():
        for t in (leaves[0], ids, dy):
            t.copy_(t.flip(0))
    graph.replay()
    other.replay()
    graph.replay()
    torch.cuda.synchronize()
    want = kq.lora_update(y, *leaves, ids, s)
    for p, q in zip((out, *grads), (want, *torch.autograd.grad(want, leaves, dy))):
        assert torch.equal(p, q)
    assert torch.equal(out2, kq.lora_update(y, x, a, b, ids, s))


def test_gradient_against_differences():
    """The gradient in the direction of the parameters themselves, from two updates in float64 arithmetic of rounded outputs: y is
    linear in b and in a, so that a difference of outputs far apart is exact up to their rounding."""
    T, K, N, r, G = 40, 96, 80, 8, 2
    y, x, a, b, s, dy = made(11, T, K, N, r, G, "f16", "f32")
    ids = torch.arange(T, device="cuda", dtype=torch.int32) % G
    zero = torch.zeros_like(y)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    grads = torch.autograd.grad(kq.lora_update(zero, *leaves, ids, s), leaves, dy)
    base = [x, a, b]
    for k, (leaf, grad) in enumerate(zip(base, grads)):
        step = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(k)).cuda().to(leaf.dtype)
        with_step, without = list(base), list(base)
        with_step[k] = step                        # linear: f(step) itself is the derivative in its direction
        moved = kq.lora_update(zero, *with_step, ids, s).double()
        lhs = (moved * dy.double()).sum()
        rhs = (grad.double() * step.double()).sum()
        # roundings: half a step of each moved output and of each gradient
        tol = 2.0 ** -11 * (moved * dy.double()).abs().sum() + (2.0 ** -11 if k == 0 else 2.0 ** -20) * (grad.double() * step.double()).abs().sum()
        assert abs(lhs - rhs) <= tol + 1e-4 * abs(lhs)


def test_offsets_beyond_32_bits():
    """A stack whose last adapter starts beyond 2^31 elements."""
    free, _ = torch.cuda.mem_get_info()
    G, r, K = 1100, 128, 16384                     # 2.3e9 elements in a
    if free < 12 << 30:
        pytest.skip("needs 12 GB")
    a = torch.zeros(G, r, K, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(G, 8, r, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    a[-1] = torch.randn(r, K, device="cuda", generator=g) * K ** -0.5
    b[-1] = torch.randn(8, r, device="cuda", generator=g) * 0.1
    x = torch.randn(3, K, device="cuda", generator=g).bfloat16()
    y = torch.zeros(3, 8, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([G - 1, 0, G - 1], device="cuda", dtype=torch.int32)
    out = kq.lora_update(y, x, a, b, ids)
    want = plain(y[::2], x[::2], a[-1:], b[-1:], np.zeros(2, int), [1.0])
    check(out[::2], want["y"])
    assert (out[1] == 0).all()


@pytest.mark.parametrize("n,slots,G,E", [(1, 1, 1, 1), (300, 3, 2, 5), (5000, 1, 3, 1), (4096, 8, 1, 128), (12288, 4, 2, 300), (33000, 8, 4, 60),
                                         (200_000, 1, 40, 1), (140_000, 7, 1, 1023), (3000, 2, 1, 2000), (9000, 9, 900, 60)])
def test_order_by_groups(n, slots, G, E):
    """The plan: entries by group and stable, where each group starts, tiles that cover all of them once."""
    from mlx_kquant_b200 import _lib
    rng = np.random.default_rng(n)
    ids = np.where(rng.random(n // slots) < 0.1, rng.choice([-1, G, 2 ** 31 - 1], n // slots), rng.integers(0, G, n // slots)).astype(np.int32)
    ex = np.where(rng.random(n) < 0.1, -1, rng.integers(0, E + 1, n)).astype(np.int32)
    L, NG = _lib.lib(), G * E
    for use_ids, use_ex in ((True, True), (True, False), (False, True)):
        if (not use_ids and G > 1) or (not use_ex and E > 1):
            continue
        plan = torch.full((L.kq_lora_plan_bytes(n, NG) + 256,), 0x5a, dtype=torch.uint8, device="cuda")
        di, de = torch.from_numpy(ids).cuda(), torch.from_numpy(ex).cuda()
        _lib.check(L.kq_lora_plan(di.data_ptr() if use_ids else None, de.data_ptr() if use_ex else None, n, slots, G, E, plan.data_ptr(),
                                  plan.numel() - 256, torch.cuda.current_stream().cuda_stream))
        got = plan.cpu().numpy()
        assert (got[-256:] == 0x5a).all()
        i, x = (np.repeat(ids, slots) if use_ids else np.zeros(n, int)), (ex if use_ex else np.zeros(n, int))
        key = np.where((i >= 0) & (i < G) & (x >= 0) & (x < E), i.astype(np.int64) * E + x, NG)
        up = lambda v: (v + 255) // 256 * 256  # noqa: E731
        order = got[:4 * n].view(np.int32)
        assert np.array_equal(order, np.argsort(key, kind="stable"))
        offsets = got[up(4 * n):up(4 * n) + 4 * (NG + 2)].view(np.int32)
        assert np.array_equal(offsets, np.concatenate([[0], np.cumsum(np.bincount(key, minlength=NG + 1))]))
        height = 64 if n > 2048 and n >= 24 * NG else 16
        at = up(up(4 * n) + 4 * (NG + 2))
        tiles = got[at:at + 16 * (n // height + NG + 1)].view(np.int32).reshape(-1, 4)
        seen = np.zeros(n, int)
        for g, start, rows, _ in tiles[tiles[:, 2] > 0]:
            assert rows <= height and (key[order[start:start + rows]] == (g if g >= 0 else NG)).all()
            seen[start:start + rows] += 1
        assert (seen == 1).all()
