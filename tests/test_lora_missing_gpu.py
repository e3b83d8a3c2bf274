"""The routed layer where a row runs out of experts (index -1, weight 0): such entries add nothing, forward and backward."""
import pytest
import torch

import mlx_kquant_b200 as kq
from mlx_kquant_b200.moe import combine, moe_router_grouped
from mlx_kquant_b200.nn import KQuantLoRASwitchLinear, KQuantSwitchLinear
from test_lora_nn_gpu import off, wire

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def unwritten_memory_is_nan():
    """torch.empty gives NaN, so that what is never written is seen."""
    was = torch.utils.deterministic.fill_uninitialized_memory
    torch.use_deterministic_algorithms(True, warn_only=True)
    torch.utils.deterministic.fill_uninitialized_memory = True
    yield
    torch.use_deterministic_algorithms(False)
    torch.utils.deterministic.fill_uninitialized_memory = was


def layer(E=6, N=72, K=256, G=2, bias=False):
    base = KQuantSwitchLinear(E, N, K, bias, "q4_k").cuda()
    base.weight.copy_(wire("q4_k", E, N, K, seed=3))
    if bias:
        base.bias.normal_(generator=torch.Generator(device="cuda").manual_seed(8))
    made = KQuantLoRASwitchLinear(base, 8, G, 0.75)
    with torch.no_grad():
        made.lora_b.copy_(torch.randn(made.lora_b.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)) * 0.1)
    return made


@pytest.mark.parametrize("T", [5, 300])
@pytest.mark.parametrize("per_slot", [False, True])
def test_rows_that_run_out_of_experts(T, per_slot):
    E, N, K, R, G = 6, 72, 256, 4, 2
    up = layer(E, N, K, G)
    g = torch.Generator(device="cuda").manual_seed(T)
    logits = torch.randn(T, E, device="cuda", generator=g)
    logits[::3, 2:] = -torch.inf
    logits[1] = -torch.inf
    logits.requires_grad_()
    ids = torch.randint(-1, G, (T,), device="cuda", generator=g, dtype=torch.int32)
    x = torch.randn(T, R if per_slot else 1, 1, K, device="cuda", generator=g).bfloat16().requires_grad_()
    idx, w = moe_router_grouped(logits, R)
    h = up(x, idx, ids)
    none = idx < 0
    assert none[1].all() and none[0].sum() == 2 and not h[none].any() and h.isfinite().all()
    y = (h.view(T, R, N).float() * w[:, :, None]).sum(1)
    dy = torch.randn(T, N, device="cuda", generator=g)
    leaves = (logits, x, up.lora_a, up.lora_b)
    got = torch.autograd.grad(y, leaves, dy)
    W = kq.dequantize(up.base.weight, up.base.scales, "q4_k", torch.float32).double()
    ld, xd, a, b = (t.detach().double().requires_grad_() for t in leaves)
    e, ad = idx.clamp(min=0).long().reshape(-1), ids.clamp(min=0).long().repeat_interleave(R)
    on, use = (~none).reshape(-1, 1).double(), (ids >= 0).double().repeat_interleave(R)[:, None]
    rows = xd.expand(T, R, 1, K).reshape(-1, K)
    s = torch.where(none, 0.0, torch.sigmoid(ld).gather(1, idx.clamp(min=0).long()))
    wd = s / (s.sum(1, keepdim=True) + 1e-20)
    d = on * (torch.einsum("tnk,tk->tn", W[e], rows) + 0.75 * use * torch.einsum("tnr,trk,tk->tn", b[ad, e], a[ad, e], rows))
    ref = (d.view(T, R, N) * wd[:, :, None]).sum(1)
    want = torch.autograd.grad(ref, (ld, xd, a, b), dy.double())
    # bf16 between the steps: two roundings forward, two back, 2^-9 rms each at most, and the products' own 2e-3
    assert off(y, ref) < 2 * 2.0 ** -9 + 2e-3
    for p, q in zip(got, want):
        assert p.isfinite().all() and off(p, torch.nan_to_num(q)) < 4 * 2.0 ** -9 + 4e-3
    with torch.no_grad():
        plain = up(x, idx, ids)
        assert torch.equal(plain, h)
        out = combine(plain.view(T * R, N).contiguous(), w.contiguous(), R)
        assert out.isfinite().all() and not out[1].any()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.uint32, torch.int16])
@pytest.mark.parametrize("grad", [False, True])
def test_indices_out_of_range(dtype, grad):
    """Below zero and beyond the stack, a bias at the experts, all types of indices, routed and flat."""
    up = layer(bias=True)
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(8, 1, 1, 256, device="cuda", generator=g).bfloat16().requires_grad_(grad)
    idx = torch.tensor([[0, 5], [6, 1], [1, 9], [3, 3], [30000, 2], [5, 0], [2, 7], [4, 4]], device="cuda")
    if dtype != torch.uint32:
        idx[0, 1], idx[5, 0] = -1, -7
    if dtype == torch.int64:
        idx[6, 1] = 2 ** 32 + 1
    ids = torch.tensor([0, 1, -1, 0, 1, 0, 1, 1], device="cuda", dtype=torch.int32)
    out = (idx < 0) | (idx >= 6)
    given = idx.to(dtype)
    y = up(x, given, ids)
    with torch.no_grad():
        good = up(x, torch.where(out, 0, idx).int(), ids)
    assert not y[out].any() and torch.equal(y[~out], good[~out])
    if grad:
        dy = torch.randn(y.shape, device="cuda", generator=g).bfloat16()
        dx, da, db = torch.autograd.grad(y, (x, up.lora_a, up.lora_b), dy)
        again = torch.autograd.grad(up(x, torch.where(out, 0, idx).int(), ids), (x, up.lora_a, up.lora_b), torch.where(out[..., None, None], 0, dy))
        for p, q in zip((dx, da, db), again):
            assert p.isfinite().all() and torch.equal(p, q)
    # flat rows in the order of their experts, as many as take the segment product
    many = torch.sort(torch.randint(-2 if dtype != torch.uint32 else 0, 8, (700,), device="cuda", generator=g)).values
    rows = torch.randn(700, 1, 256, device="cuda", generator=g).bfloat16().requires_grad_(grad)
    of = torch.randint(0, 2, (700,), device="cuda", generator=g, dtype=torch.int32)
    y = up(rows, many.to(dtype), of, sorted_indices=True)
    out = (many < 0) | (many >= 6)
    assert out.any() and not y[out].any() and y.isfinite().all() and y[~out].any(-1).all()


@pytest.mark.parametrize("T,R,N", [(1, 1, 8), (5, 3, 7), (700, 8, 1001), (64, 1, 40000)])
def test_clear_rows(T, R, N):
    """All rows of indices outside the stack, to their ends, and no others; rows that start anywhere."""
    from mlx_kquant_b200 import _lib
    g = torch.Generator(device="cuda").manual_seed(T)
    for skip in (0, 1, 8):
        buf = torch.randn(T * R * N + 16, device="cuda", generator=g).half()
        was = buf.clone()
        idx = torch.randint(-1, 4, (T, R), device="cuda", generator=g, dtype=torch.int32)
        _lib.check(_lib.lib().kq_clear_rows(buf.data_ptr() + 2 * skip, T * R, N, idx.data_ptr(), 3, torch.cuda.current_stream().cuda_stream))
        want = was.clone()
        want[skip:skip + T * R * N].view(T * R, N)[((idx < 0) | (idx > 2)).view(-1)] = 0
        assert torch.equal(buf, want)


def test_host_rows_are_refused():
    up = layer()
    with pytest.raises(RuntimeError, match="CUDA device"):
        up(torch.zeros(2, 1, 1, 256), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
