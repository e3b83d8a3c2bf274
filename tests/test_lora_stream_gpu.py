"""Calls on a given stream: their operands stay theirs until the kernels there have run, even if the caller drops them at once."""
import pytest
import torch

import mlx_kquant_b200 as kq
from mlx_kquant_b200.moe import gather_lora_update
from test_lora_gpu import made, some_ids
from test_lora_nn_gpu import wire

pytestmark = pytest.mark.gpu


def held_up():
    """A stream with some 50 ms of work ahead."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    return side


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("T", [6, 40, 300])
def test_composed_product_drops_its_operands(T, ids_dtype):
    K, N, r, G = 512, 96, 8, 3
    w = wire("q4_k", N, K, seed=1)
    _, x, a, b, s, _ = made(T, T, K, N, r, G, "bf16", "bf16")
    ids = torch.from_numpy(some_ids(T, T, G)).cuda().to(ids_dtype)
    want = kq.quantized_matmul_lora(x, w, None, "q4_k", a, b, ids, s)
    torch.cuda.synchronize()
    side = held_up()
    given = [t.clone() for t in (a, b, ids, s)]
    shapes = [(t.shape, t.dtype) for t in given]
    out = kq.quantized_matmul_lora(x.float() if T == 40 else x.clone(), w, None, "q4_k", *given, stream=side)
    del given
    # the allocator gives the same memory to the next tensors of these sizes, unless it knows better
    others = [torch.full(shape, 1, dtype=dtype, device="cuda") for shape, dtype in shapes * 2]
    others += [torch.full((T, K), 7.0, dtype=d, device="cuda") for d in (torch.bfloat16, torch.float32) * 2]
    torch.cuda.synchronize()
    assert torch.equal(out, want) and len(others) == 12


@pytest.mark.parametrize("T", [6, 300])
def test_updates_drop_their_operands(T):
    y, x, a, b, s, _ = made(T, T, 64, 40, 8, 2, "bf16", "bf16", E=3, slots=2)
    ids = torch.from_numpy(some_ids(T, T, 2)).cuda()
    idx = torch.randint(-1, 3, (T, 2), device="cuda")
    for op, args in ((kq.lora_update, (y[:, 0], x, a[:, 0], b[:, 0], ids.long(), s.double())), (gather_lora_update, (y, x, a, b, idx, ids, s))):
        want = op(*args)
        torch.cuda.synchronize()
        side = held_up()
        given = [t.clone() for t in args]
        shapes = [(t.shape, t.dtype) for t in given]
        out = op(*given, stream=side)
        del given
        others = [torch.full(shape, 1, dtype=dtype, device="cuda") for shape, dtype in shapes * 2]
        torch.cuda.synchronize()
        assert torch.equal(out, want) and others
