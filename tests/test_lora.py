"""Low-rank adapters without a GPU: what is refused, and with which words."""
import pytest
import torch

import mlx_kquant_b200 as kq
from mlx_kquant_b200 import _lib
from mlx_kquant_b200.moe import gather_lora_update

BF = torch.bfloat16


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def test_refusals():
    y, x, a, b = z(4, 6), z(4, 8), z(2, 3, 8), z(2, 6, 3)
    ids = torch.zeros(4, dtype=torch.int32)
    for args, words in (
        ((y.float(), x, a, b, ids), "float16 or bfloat16"),
        ((y, x.half(), a, b, ids), "x must be of y's dtype"),
        ((y.half(), x.float(), a.half(), b.half(), ids), "x must be of y's dtype"),
        ((y, x, a.half(), b.half(), ids), "y's dtype or float32"),
        ((y, x, a, b.float(), ids), "y's dtype or float32"),
        ((y, x, z(2, 129, 8), z(2, 6, 129), ids), "rank must be 1 to 128"),
        ((y, x, z(2, 0, 8), z(2, 6, 0), ids), "rank must be 1 to 128"),
        ((y, x, a, z(2, 5, 3), ids), "do not fit"),
        ((y, x, z(2, 3, 7), b, ids), "do not fit"),
        ((y, x, z(1, 3, 8), b, ids), "do not fit"),
        ((y, z(5, 8), a, b, ids), "same rows"),
        ((y, x, a, b), "need adapter_ids"),
        ((y, x, a, b, ids[:3]), "leading axes"),
        ((y, x, a, b, ids.float()), "leading axes"),
        ((y, x, a[0, 0], b, ids), "must be \\[adapters, r, K\\]"),
    ):
        with pytest.raises(ValueError, match=words):
            kq.lora_update(*args)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kq.lora_update(y, x, a, b, ids)


def test_refusals_beside_experts():
    y, x, a, b = z(4, 2, 6), z(4, 8), z(2, 5, 3, 8), z(2, 5, 6, 3)
    idx, ids = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for args, words in (
        ((y, x, a, b, idx), "need adapter_ids"),
        ((y, z(3, 8), a, b, idx, ids), "x must be"),
        ((y, z(4, 3, 8), a, b, idx, ids), "x must be"),
        ((y[:, :1], x, a, b, idx, ids), "indices \\[T, R\\]"),
        ((y, x, a, b, idx[0], ids), "indices \\[T, R\\]"),
        ((y, x, a, b, idx.float(), ids), "integers"),
        ((y, x, a, b, idx, idx), "integers of shape"),
        ((y, x, a[0, 0], b, idx, ids), "must be \\[adapters, experts, r, K\\]"),
        ((y, x, a, z(2, 4, 6, 3), idx, ids), "do not fit"),
        ((y, x, z(2, 40000, 1, 8), z(2, 40000, 6, 1), idx, ids), "65535"),
    ):
        with pytest.raises(ValueError, match=words):
            gather_lora_update(*args)
    with pytest.raises(RuntimeError, match="no CPU path"):
        gather_lora_update(y, x, a, b, idx, ids)


def test_c_entries_refuse_before_touching_memory():
    L, F16, BF16, F32, bad = _lib.lib(), _lib.KQ_F16, _lib.KQ_BF16, _lib.KQ_F32, _lib.KQ_ERR_INVALID_ARGUMENT
    p = 256   # never followed

    def update(dtype=F16, rows=4, K=8, slots=1, pt=F16, rank=2, N=8, G=2, E=1, ids=p, experts=None, plan=None, plan_bytes=0, x=p):
        return L.kq_lora_update(x, dtype, rows, K, K, slots, 0, p, p, pt, rank, N, G, E, ids, experts, None, 1.0, p, N, p, N, None,
                                plan, plan_bytes, None)

    for kw in (dict(dtype=F32), dict(pt=BF16), dict(dtype=BF16, pt=F16), dict(rank=0), dict(rank=129), dict(rows=-1), dict(rows=5, slots=2),
               dict(slots=0), dict(rows=2 ** 31), dict(G=0), dict(G=65535, E=2, experts=p), dict(ids=None), dict(K=0), dict(N=0),
               dict(plan=p, plan_bytes=16), dict(x=None)):
        assert update(**kw) == bad, kw
        assert b"[mlx_kquant.lora_update]" in L.kq_last_error()
    assert update(rows=0) == 0
    need = L.kq_lora_plan_bytes(1000, 8)
    assert need > 1000 * 4 and L.kq_lora_plan_bytes(-1, 8) == 0 and L.kq_lora_plan_bytes(10, 0) == 0
    assert L.kq_lora_plan(p, None, 1000, 1, 8, 1, p, need - 1, None) == bad
    assert L.kq_lora_backward_workspace_bytes(64, 1, 0, 4096, 4096, 16, F16) >= L.kq_lora_saved_bytes(64, 16, F16) == 64 * 16 * 4
    back = lambda ids=p, plan=None, ws=0: L.kq_lora_backward(  # noqa: E731
        p, F16, 4, 8, 8, p, 8, 8, 1, 0, p, p, F16, 2, 2, 1, ids, None, None, 1.0, p, p, p, p, plan, 1 << 20, p, ws, None)
    assert back() == bad and b"plan" in L.kq_last_error()
    assert back(plan=p) == bad and b"workspace" in L.kq_last_error()
