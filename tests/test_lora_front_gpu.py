"""The native front of lora_update, gather_lora_update and moe_router_grouped against the Python form of the same calls."""
import pytest
import torch

import mlx_kquant_b200 as kq
from mlx_kquant_b200 import _lib, lora, moe

pytestmark = pytest.mark.gpu


def both(monkeypatch, call):
    """The call as it is, and with the front out of the way; an exception counts as an outcome."""
    def outcome():
        try:
            return call()
        except Exception as e:
            return type(e), str(e)
    here = outcome()
    with monkeypatch.context() as m:
        m.setattr(lora, "_front_lora", lambda *args: None)
        m.setattr(moe, "_front_route", lambda *args: None)
        return here, outcome()


def same(a, b):
    if isinstance(a, tuple):
        return type(b) is tuple and len(a) == len(b) and all(same(p, q) for p, q in zip(a, b))
    if not isinstance(a, torch.Tensor):
        return a == b
    return (a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype and a.device == b.device
            and a.requires_grad == b.requires_grad and torch.equal(a, b))


@pytest.mark.parametrize("T", [1, 9, 150])
def test_update(monkeypatch, T):
    g = torch.Generator(device="cuda").manual_seed(T)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, y, a, b = rnd(T, 64).half(), rnd(T, 40).half(), (rnd(3, 8, 64) * 0.1).half(), (rnd(3, 40, 8) * 0.1).half()
    ids = torch.randint(-1, 4, (T,), device="cuda", generator=g, dtype=torch.int32)
    s = torch.rand(3, device="cuda", generator=g)
    front = _lib.torch_front()
    assert isinstance(front.lora(y, x, a, b, ids, s, None, 128), torch.Tensor)
    assert front.lora(y, x, a, b, None, s, None, 128) is None and front.lora(y.cpu(), x, a, b, ids, s, None, 128) is None
    calls = [(y, x, a, b, ids, s), (y, x, a.float(), b.float(), ids, s), (y, x, a, b, ids, 0.5), (y, x, a, b, ids, None), (y, x, a, b, ids, 2),
             (y, x, a, b, ids.long(), s), (y, x, a[1], b[1], None, None), (y, x, a[:1], b[:1]), (y, x, a, b), (y, x, a, b, ids[:0], s),
             (y, x.float(), a, b, ids, s), (y.bfloat16(), x.float(), a.bfloat16(), b.bfloat16(), ids, s), (y, x, a, b.float(), ids, s),
             (y[None], x[None], a, b, ids[None], s), (y[None], x[None], a, b, ids[:1], s), (y[0], x[0], a[0], b[0]), (y[:0], x[:0], a, b, ids[:0], s),
             (y, x, a.transpose(1, 2).contiguous().transpose(1, 2), b, ids, s), (y, x, a, b, ids, s[:2]), (y, x, a, b, ids, s.double()),
             (y, x[:, :32], a, b, ids, s), (y, torch.nn.Parameter(x), a, b, ids, s), (y.cpu(), x, a, b, ids, s), (y, x, a, b, ids.float(), s)]
    for c in calls:
        p, q = both(monkeypatch, lambda: kq.lora_update(*c))
        assert same(p, q), [getattr(t, "shape", t) for t in c]
    with torch.no_grad():
        p, q = both(monkeypatch, lambda: kq.lora_update(y, torch.nn.Parameter(x), a, b, ids, s))
        assert same(p, q) and isinstance(p, torch.Tensor)


def test_update_beside_experts(monkeypatch):
    g = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    for T in (5, 60):
        x, y, a, b = rnd(T, 64).half(), rnd(T, 3, 40).half(), (rnd(2, 6, 8, 64) * 0.1).half(), (rnd(2, 6, 40, 8) * 0.1).half()
        idx = torch.randint(-1, 7, (T, 3), device="cuda", generator=g, dtype=torch.int32)
        ids = torch.randint(-1, 3, (T,), device="cuda", generator=g, dtype=torch.int32)
        for c in [(y, x, a, b, idx, ids), (y, x[:, None].repeat(1, 3, 1), a, b, idx, ids, 0.5), (y, x, a, b, idx.long(), ids), (y, x, a[0], b[0], idx),
                  (y, x, a[:1], b[:1], idx), (y, x, a, b, idx), (y, x, a, b, idx[:, :2], ids), (y, x, a, b, idx, idx), (y, x, a, b, idx.T, ids),
                  (y.transpose(0, 1).contiguous().transpose(0, 1), x, a, b, idx, ids)]:
            p, q = both(monkeypatch, lambda: moe.gather_lora_update(*c))
            assert same(p, q), [getattr(t, "shape", t) for t in c]


def test_router(monkeypatch):
    g = torch.Generator(device="cuda").manual_seed(6)
    x, bias = torch.randn(7, 64, device="cuda", generator=g), torch.randn(64, device="cuda", generator=g)
    for args, kw in [((x, 4), {}), ((x, 4, 8, 3), dict(bias=bias)), ((x.half(), 4, 8, 3), dict(scoring="softmax", group_top=1)),
                     ((x, 4), dict(norm_topk_prob=False, scale=2.5)), ((x, 4), dict(norm_topk_prob=1, scale=2)), ((x[:, ::2], 4), {}), ((x[:0], 4), {}),
                     ((x, 4), dict(bias=bias.double())), ((x, 4), dict(bias=bias[:3])), ((x, 4), dict(bias=torch.nn.Parameter(bias))), ((x, 65), {}),
                     ((x, 4, 7), {}), ((x, 4, 8, 9), {}), ((x, 20, 8, 1), {}), ((x, 4), dict(group_top=3)), ((x, 4), dict(scoring="tanh")),
                     ((x.double(), 4), {}), ((x[0], 4), {}), ((torch.nn.Parameter(x), 4), {}), ((x.cpu(), 4), {})]:
        p, q = both(monkeypatch, lambda: moe.moe_router_grouped(*args, **kw))
        if isinstance(p, tuple) and isinstance(p[0], type):
            assert q[0] is p[0], (p, q)          # refused by both, as one kind of error
        else:
            assert same(p, q), kw


@pytest.mark.parametrize("T", [5, 200])
def test_gradients(monkeypatch, T):
    g = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    ids = torch.randint(-1, 4, (T,), device="cuda", generator=g, dtype=torch.int32)
    idx = torch.randint(-1, 6, (T, 3), device="cuda", generator=g, dtype=torch.int32)
    y, x, a, b = rnd(T, 40).bfloat16(), rnd(T, 64).bfloat16(), rnd(3, 8, 64) * 0.1, rnd(3, 40, 8) * 0.1
    y3, a4, b4 = rnd(T, 3, 40).bfloat16(), rnd(3, 6, 8, 64) * 0.1, rnd(3, 6, 40, 8) * 0.1
    logits, bias = rnd(T, 64), rnd(64) * 0.1

    def step(op, leaves, want, *rest):
        leaves = [t.detach().clone().requires_grad_(w) for t, w in zip(leaves, want)]
        out = op(*leaves, *rest)
        out = out[1] if isinstance(out, tuple) else out
        assert out.requires_grad
        dy = torch.ones(1, device="cuda", dtype=out.dtype).expand(out.shape)   # not contiguous
        return (out.detach(), *torch.autograd.grad(out, [t for t in leaves if t.requires_grad], dy))

    for want in ((1, 1, 1, 1), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 0, 0)):
        p, q = both(monkeypatch, lambda: step(kq.lora_update, (y, x, a, b), want, ids, None))
        assert same(p, q), want
        p, q = both(monkeypatch, lambda: step(moe.gather_lora_update, (y3, x, a4, b4), want, idx, ids, 0.5))
        assert same(p, q), want
    p, q = both(monkeypatch, lambda: step(lambda l: moe.moe_router_grouped(l, 4, 8, 3, bias=bias), (logits,), (1,)))
    assert same(p, q)
    # a second gradient is refused by both
    for call in (lambda: step2(kq.lora_update, a, lambda t: (y, x, t, b, ids)), lambda: step2(moe.moe_router_grouped, logits, lambda t: (t, 4))):
        for out in both(monkeypatch, call):
            assert isinstance(out, tuple) and out[0] is RuntimeError, out


def step2(op, leaf, args):
    leaf = leaf.detach().clone().requires_grad_()
    out = op(*args(leaf))
    out = out[1] if isinstance(out, tuple) else out
    first, = torch.autograd.grad(out.float().square().sum(), leaf, create_graph=True)
    return torch.autograd.grad(first.square().sum(), leaf)
