"""What the C entries of the low-rank adapters and the grouped router refuse before any launch: operands off their alignment, long calls
without an order of their entries."""
import pytest

from mlx_kquant_b200 import _lib

L, F16, F32, BAD = _lib.lib(), _lib.KQ_F16, _lib.KQ_F32, _lib.KQ_ERR_INVALID_ARGUMENT
P = 1 << 20   # never followed


def update(rows=4, x=P, a=P, b=P, pt=F16, ids=P, experts=None, scaling=None, y=P, out=P, saved=None, plan=None, plan_bytes=1 << 30):
    return L.kq_lora_update(x, F16, rows, 8, 8, 1, 0, a, b, pt, 2, 8, 2, 1, ids, experts, scaling, 1.0, y, 8, out, 8, saved, plan, plan_bytes, None)


def backward(dy=P, x=P, a=P, b=P, pt=F16, scaling=None, saved=P, dx=P, da=P, db=P, plan=P, ws=P):
    return L.kq_lora_backward(dy, F16, 4, 8, 8, x, 8, 8, 1, 0, a, b, pt, 2, 2, 1, P, None, scaling, 1.0, saved, dx, da, db, plan, 1 << 30, ws, 1 << 30, None)


@pytest.mark.parametrize("kw", [dict(plan=P + 16), dict(plan=P + 128), dict(saved=P + 8), dict(saved=P + 2), dict(x=P + 1), dict(y=P + 1), dict(out=P + 1),
                                dict(a=P + 1), dict(b=P + 1), dict(a=P + 2, pt=F32), dict(b=P + 2, pt=F32), dict(ids=P + 2), dict(experts=P + 1),
                                dict(scaling=P + 2)], ids=str)
def test_update_off_alignment(kw):
    assert update(**kw) == BAD and b"[mlx_kquant.lora_update]" in L.kq_last_error() and b"aligned" in L.kq_last_error()


@pytest.mark.parametrize("kw", [dict(plan=P + 16), dict(saved=P + 8), dict(ws=P + 128), dict(dy=P + 1), dict(x=P + 1), dict(dx=P + 1), dict(da=P + 1),
                                dict(db=P + 1), dict(db=P + 2, pt=F32), dict(a=P + 2, pt=F32), dict(b=P + 1), dict(scaling=P + 1)], ids=str)
def test_backward_off_alignment(kw):
    assert backward(**kw) == BAD and b"[mlx_kquant.lora_backward]" in L.kq_last_error() and b"aligned" in L.kq_last_error()


def test_plan_off_alignment():
    for kw in ((P + 16, P, None), (P, P + 2, None), (P, P, P + 2)):
        assert L.kq_lora_plan(kw[1], kw[2], 4, 1, 2, 1, kw[0], 1 << 30, None) == BAD and b"aligned" in L.kq_last_error()


def test_router_off_alignment():
    fwd = lambda logits=P, bias=P, idx=P, w=P, dt=F16: L.kq_moe_router_grouped(logits, dt, 2, 16, 2, 1, 1, 1, b"sigmoid", bias, 1, 1.0, idx, w, None)  # noqa: E731
    for kw in (dict(logits=P + 1), dict(logits=P + 2, dt=F32), dict(bias=P + 2), dict(idx=P + 2), dict(w=P + 1)):
        assert fwd(**kw) == BAD and b"[mlx_kquant.moe_router_grouped]" in L.kq_last_error() and b"aligned" in L.kq_last_error(), kw
    back = lambda logits=P, idx=P, dw=P, dl=P: L.kq_moe_router_grouped_backward(logits, F16, 2, 16, 2, b"sigmoid", 1, 1.0, idx, dw, dl, None)  # noqa: E731
    for kw in (dict(logits=P + 1), dict(idx=P + 1), dict(dw=P + 2), dict(dl=P + 1)):
        assert back(**kw) == BAD and b"aligned" in L.kq_last_error(), kw


def test_clear_rows():
    call = lambda y=P, rows=4, n=8, experts=P, E=2: L.kq_clear_rows(y, rows, n, experts, E, None)  # noqa: E731
    for kw in (dict(y=None), dict(experts=None), dict(rows=-1), dict(rows=2 ** 30 + 1), dict(n=0), dict(E=0), dict(y=P + 1), dict(experts=P + 2)):
        assert call(**kw) == BAD and b"[mlx_kquant.clear_rows]" in L.kq_last_error(), kw
    assert call(rows=0) == 0


def test_long_calls_need_the_order_of_their_entries():
    for rows in (65537, 2 ** 24, 2 ** 29 + 1, 2 ** 30):
        assert update(rows=rows) == BAD and b"plan" in L.kq_last_error()
