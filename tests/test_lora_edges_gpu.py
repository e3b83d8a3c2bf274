"""Low-rank adapters: tall tiles, empty batches with gradients, expanded rows, overlapping outputs, index types."""
import pytest
import torch

import mlx_kquant_b200 as kq
from lora_plain import check, group_list, plain
from mlx_kquant_b200 import lora
from mlx_kquant_b200.moe import gather_lora_update
from test_lora_gpu import TYPES, made, some_ids

pytestmark = pytest.mark.gpu

# enough rows for tiles of 64, of one adapter and of several: odd lengths, ranks of every template, a last tile of one row
TALL = [(1409, 96, 264, 24, 1), (1345, 33, 17, 3, 1), (2112, 136, 72, 128, 3), (2200, 100, 129, 33, 2), (2500, 1024, 96, 64, 7), (2113, 72, 100, 5, 40)]


@pytest.fixture(params=["front", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(lora, "_front_lora", lambda *a: None)
    return request.param


@pytest.mark.parametrize("size", TALL, ids=str)
@pytest.mark.parametrize("dt,pt", TYPES)
def test_tall_tiles(size, dt, pt):
    T, K, N, r, G = size
    y, x, a, b, s, dy = made(sum(size), T, K, N, r, G, dt, pt)
    ids = some_ids(T, T, G) if G > 1 else None
    dev_ids = None if ids is None else torch.from_numpy(ids).cuda()
    want = plain(y, x, a, b, group_list(ids, 1, None, G, 1, T), s.cpu().numpy(), dy=dy)
    check(kq.lora_update(y, x, a, b, dev_ids, s), want["y"], "y")
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    got = torch.autograd.grad(kq.lora_update(y, *leaves, dev_ids, s), leaves, dy)
    for name, g in zip(("dx", "da", "db"), got):
        check(g, want[name], name)


def test_tall_tiles_of_rows_without_an_adapter():
    y, x, a, b, s, _ = made(5, 2300, 64, 100, 8, 3, "bf16", "bf16")
    ids = torch.from_numpy(some_ids(9, 2300, 3)).cuda()
    ids[200:1700] = -1
    x[200:1700] = torch.inf
    out = kq.lora_update(y, x, a, b, ids, s)
    none = (ids < 0) | (ids >= 3)
    assert torch.equal(out[none], y[none]) and out[~none].isfinite().all() and not torch.equal(out[~none], y[~none])


def gradients_are_zero(out, leaves):
    got = torch.autograd.grad(out.float().sum(), leaves)
    for t, g in zip(leaves, got):
        assert g.shape == t.shape and g.dtype == t.dtype and not g.any()


@pytest.mark.parametrize("ids", [False, True])
def test_an_empty_batch_has_gradients(path, ids):
    y, x, a, b, s, _ = made(1, 3, 64, 40, 8, 2 if ids else 1, "bf16", "f32")
    leaves = [t.requires_grad_() for t in (y[:0].detach(), x[:0].detach(), a, b)]
    out = kq.lora_update(*leaves, torch.zeros(0, dtype=torch.int32, device="cuda") if ids else None, s)
    assert out.shape == (0, 40) and out.requires_grad
    gradients_are_zero(out, leaves)
    out = kq.lora_update(y[:0].detach(), x[:0].detach(), a.detach(), b, torch.zeros(0, dtype=torch.int32, device="cuda") if ids else None, s)
    gradients_are_zero(out, [b])


@pytest.mark.parametrize("shape", [(0, 3), (4, 0)])
def test_no_slots_have_gradients(path, shape):
    T, R = shape
    _, _, a, b, s, _ = made(2, 1, 64, 40, 8, 2, "bf16", "bf16", E=3)
    y, x = (torch.zeros(T, *d, dtype=torch.bfloat16, device="cuda").requires_grad_() for d in ((R, 40), (64,)))
    leaves = [y, x, a.requires_grad_(), b.requires_grad_()]
    out = gather_lora_update(*leaves, torch.zeros(T, R, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda"), s)
    assert out.shape == (T, R, 40)
    gradients_are_zero(out, leaves)


@pytest.mark.parametrize("T", [6, 300])
def test_rows_of_one_tensor(path, T):
    """x and the incoming gradient are one row, expanded: strides of zero."""
    y, x, a, b, s, dy = made(T, T, 64, 48, 8, 2, "bf16", "f32")
    ids = some_ids(T, T, 2)
    dev_ids = torch.from_numpy(ids).cuda()
    x1, d1 = x[:1].expand(T, -1), dy[:1].expand(T, -1)
    want = plain(y, x1, a, b, group_list(ids, 1, None, 2, 1, T), s.cpu().numpy(), dy=d1)
    leaves = [x1.detach().requires_grad_(), a.requires_grad_(), b.requires_grad_()]
    out = kq.lora_update(y, *leaves, dev_ids, s)
    check(out, want["y"], "y")
    for name, g in zip(("dx", "da", "db"), torch.autograd.grad(out, leaves, d1)):
        check(g, want[name], name)


def test_outputs_that_overlap_are_refused():
    y, x, a, b, s, _ = made(3, 9, 48, 48, 8, 1, "bf16", "bf16")
    all_rows = torch.cat([y, y[:2]])
    with pytest.raises(ValueError, match="overlap"):
        kq.lora_update(y, x, a, b, None, s, out=x)
    with pytest.raises(ValueError, match="overlap"):
        kq.lora_update(all_rows[:9], x, a, b, None, s, out=all_rows[2:])
    with pytest.raises(ValueError, match="overlap"):
        kq.lora_update(y[:8], x[:8], a, b, None, s, out=a[0])
    # the two that are meant: y itself, and its neighbour in one buffer
    want = kq.lora_update(y, x, a, b, None, s)
    both = torch.cat([y, torch.zeros_like(y)])
    assert torch.equal(kq.lora_update(both[:9], x, a, b, None, s, out=both[9:]), want) and torch.equal(both[:9], y)
    assert torch.equal(kq.lora_update(y, x, a, b, None, s, out=y), want)


@pytest.mark.parametrize("dtype", [torch.uint64, torch.complex64, torch.float32, torch.bool])
def test_indices_of_other_types_are_refused(dtype):
    y, x, a, b, s, _ = made(4, 3, 64, 40, 8, 2, "bf16", "bf16", E=3, slots=2)
    ids, idx = torch.zeros(3, dtype=dtype, device="cuda"), torch.zeros(3, 2, dtype=dtype, device="cuda")
    good = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="adapter_ids must be integers"):
        kq.lora_update(y[:, 0], x, a[:, 0], b[:, 0], ids, s)
    with pytest.raises(ValueError, match="adapter_ids must be integers"):
        gather_lora_update(y, x, a, b, torch.zeros(3, 2, dtype=torch.int32, device="cuda"), ids, s)
    with pytest.raises(ValueError, match="indices must be integers"):
        gather_lora_update(y, x, a, b, idx, good, s)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int16, torch.int8, torch.uint8, torch.uint16, torch.uint32])
def test_indices_of_all_integers(dtype):
    y, x, a, b, s, _ = made(4, 5, 64, 40, 8, 2, "bf16", "bf16")
    ids = torch.tensor([1, 0, 1, 9, 0], device="cuda")
    assert torch.equal(kq.lora_update(y, x, a, b, ids.to(dtype), s), kq.lora_update(y, x, a, b, ids.int(), s))


def layers(K=256, N=64, E=3):
    from test_lora_nn_gpu import wire
    from mlx_kquant_b200.nn import KQuantLinear, KQuantLoRALinear, KQuantLoRASwitchLinear, KQuantSwitchLinear
    one, many = KQuantLinear(K, N, False, "q8_0").cuda(), KQuantSwitchLinear(E, N, K, False, "q8_0").cuda()
    one.weight.copy_(wire("q8_0", N, K, seed=1))
    many.weight.copy_(wire("q8_0", E, N, K, seed=2))
    made = KQuantLoRALinear(one, 4, 2), KQuantLoRASwitchLinear(many, 4, 2)
    with torch.no_grad():
        for m in made:
            m.lora_b.normal_()
    return made


@pytest.mark.parametrize("T", [0, 5])
def test_layers_of_empty_batches_and_expanded_gradients(T):
    one, many = layers()
    ids = torch.ones(T, dtype=torch.int32, device="cuda")
    for layer, x, args in ((one, torch.randn(T, 256, device="cuda"), (ids,)),
                           (many, torch.randn(T, 1, 1, 256, device="cuda"), (torch.ones(T, 2, dtype=torch.int32, device="cuda"), ids))):
        for need in (True, False):
            x = x.bfloat16().detach().requires_grad_(need)
            leaves = [layer.lora_a, layer.lora_b] + [x] * need
            out = layer(x, *args)
            assert out.shape[0] == T and out.shape[-1] == 64
            d = torch.randn_like(out[:1]) if T else out.detach()
            got = torch.autograd.grad(out, leaves, d.expand(out.shape), retain_graph=True)
            want = torch.autograd.grad(out, leaves, d.expand(out.shape).contiguous())
            for p, q, t in zip(got, want, leaves):
                assert p.shape == t.shape and torch.equal(p, q)
                assert bool(p.any()) == (T > 0)
