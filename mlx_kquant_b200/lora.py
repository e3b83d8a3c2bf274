"""Low-rank adapters of many requests at once beside a shared projection (`lora_update`, `quantized_matmul_lora`) and beside an
expert stack (`moe.gather_lora_update`), with their gradients.

Adapter g of a projection [N, K] is a pair a[g] [r, K], b[g] [N, r]; a row x of a request that uses it gets
``y + s[g] * (x @ a[g].T) @ b[g].T`` on top of the projection's y. The rows of a batch may all use different adapters, and some
none. All arithmetic happens in the CUDA library (kq_lora_update, kq_lora_backward in include/kquant_b200.h): float32 sums, one
rounding to y's dtype, and between the two products x @ a.T (in the gradient dy @ b) with 16 bits, float32 parameters likewise in the
second of them. What an infinity among the operands reaches is infinite or NaN.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import KQ_BF16, KQ_F16, KQ_F32, check
from .ops import _on_device, _order_on, _stream_ptr, quantized_matmul

_DT = {torch.float32: KQ_F32, torch.float16: KQ_F16, torch.bfloat16: KQ_BF16}
MAX_RANK = 128
# up to here the update finds the rows of each adapter itself, without a launch that orders them
DIRECT_ROWS = 128


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as [rows, columns] with dense columns: a view where its strides allow."""
    r = t.reshape(-1, t.shape[-1])
    return r if r.stride(1) == 1 or r.shape[1] == 1 and r.is_contiguous() else r.contiguous()


def _integers(t: torch.Tensor) -> bool:
    return t.dtype in (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8, torch.uint16, torch.uint32)


def _overlap(t: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether the bytes from t's first to its last meet the contiguous out's."""
    if t.numel() == 0 or out.numel() == 0:
        return False
    t0, o0 = t.data_ptr(), out.data_ptr()
    t1 = t0 + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size()
    return t0 < o0 + out.numel() * out.element_size() and o0 < t1


def _refuse_tangents(op, *tensors) -> None:
    """Forward-mode differentiation, for which there is no rule: a tangent would be left out in silence."""
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"[mlx_kquant.{op}] has no forward-mode derivative; differentiate it backwards.")


def _i32(t: torch.Tensor, device) -> torch.Tensor:
    if t.dtype == torch.int64:   # (not wrapped around: what is out of range stays out of range)
        t = t.clamp(-1, 2 ** 31 - 1)
    return t.to(device=device, dtype=torch.int32).contiguous()


class _Call:
    """What the kernels are told about a call, besides the tensors that carry gradients."""

    __slots__ = ("slots", "shared", "n_adapters", "n_experts", "ids", "experts", "scaling", "scale", "stream")

    def groups(self):
        return self.n_adapters * self.n_experts

    def grouped(self):
        return self.ids is not None or self.experts is not None

    def plan(self, rows, device):
        """The entries in the order of their groups, or None where there is one group."""
        if not self.grouped():
            return None
        L = _lib.lib()
        plan = torch.empty(L.kq_lora_plan_bytes(rows, self.groups()), dtype=torch.uint8, device=device)
        _order_on(self.stream, device, plan, self.ids, self.experts)
        with _on_device(device):
            check(L.kq_lora_plan(_ptr(self.ids), _ptr(self.experts), rows, self.slots, self.n_adapters, self.n_experts,
                                 plan.data_ptr(), plan.numel(), _stream_ptr(self.stream, device)))
        return plan

    def forward(self, y, x, a, b, out, u, plan):
        yr, xr = _rows(y), _rows(x)
        a, b = a.contiguous(), b.contiguous()
        orr = out.view(-1, out.shape[-1])
        dev = x.device
        _order_on(self.stream, dev, yr, xr, a, b, out, u, plan, self.ids, self.experts, self.scaling)
        with _on_device(dev):
            check(_lib.lib().kq_lora_update(
                xr.data_ptr(), _DT[x.dtype], yr.shape[0], xr.shape[1], xr.stride(0), self.slots, int(self.shared), a.data_ptr(),
                b.data_ptr(), _DT[a.dtype], a.shape[-2], b.shape[-2], self.n_adapters, self.n_experts, _ptr(self.ids),
                _ptr(self.experts), _ptr(self.scaling), self.scale, yr.data_ptr(), yr.stride(0), orr.data_ptr(), orr.stride(0),
                _ptr(u), _ptr(plan), plan.numel() if plan is not None else 0, _stream_ptr(self.stream, dev)))

    def backward(self, dy, x, a, b, u, plan, need_x, need_a, need_b):
        dyr, xr = _rows(dy), _rows(x)
        a, b = a.contiguous(), b.contiguous()
        dev = x.device
        rows, K, r = dyr.shape[0], xr.shape[1], a.shape[-2]
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        da = torch.empty_like(a) if need_a else None
        db = torch.empty_like(b) if need_b else None
        L = _lib.lib()
        ws = torch.empty(max(256, L.kq_lora_backward_workspace_bytes(rows, self.slots, int(self.shared), K, b.shape[-2], r, _DT[a.dtype])),
                         dtype=torch.uint8, device=dev)
        with _on_device(dev):
            check(L.kq_lora_backward(
                dyr.data_ptr(), _DT[x.dtype], rows, dyr.shape[1], dyr.stride(0), xr.data_ptr(), K, xr.stride(0), self.slots,
                int(self.shared), a.data_ptr(), b.data_ptr(), _DT[a.dtype], r, self.n_adapters, self.n_experts, _ptr(self.ids),
                _ptr(self.experts), _ptr(self.scaling), self.scale, _ptr(u), _ptr(dx), _ptr(da), _ptr(db), _ptr(plan),
                plan.numel() if plan is not None else 0, ws.data_ptr(), ws.numel(), _stream_ptr(None, dev)))
        return dx, da, db


def _first_lora(*args):
    """The first call of _front_lora: the native front takes its place, or a stand-in where there is none."""
    global _front_lora
    front = _lib.torch_front()
    _front_lora = front.lora if front is not None else lambda *args: None
    return _front_lora(*args)


_front_lora = _first_lora


def front_update(y, x, a, b, adapter_ids, scaling, indices):
    """The usual call without gradients, in one native call, or None: not for that path."""
    out = _front_lora(y, x, a, b, adapter_ids, scaling, indices, DIRECT_ROWS)
    if type(out) is int:
        check(out)
    return out


class _Update(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, y, x, a, b):
        rows = y.numel() // y.shape[-1]
        plan = call.plan(rows, x.device)
        u = torch.empty(_lib.lib().kq_lora_saved_bytes(rows, a.shape[-2], _DT[a.dtype]), dtype=torch.uint8, device=x.device)
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
        call.forward(y, x, a, b, out, u, plan)
        ctx.call = call
        ctx.save_for_backward(x, a, b, u, plan, call.ids, call.experts, call.scaling)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, a, b, u, plan, *_ = ctx.saved_tensors
        _, need_y, need_x, need_a, need_b = ctx.needs_input_grad
        dx = da = db = None
        if need_x or need_a or need_b:
            dx, da, db = ctx.call.backward(dy, x, a, b, u, plan, need_x, need_a, need_b)
        return None, dy if need_y else None, dx, da, db


class _Empty(torch.autograd.Function):
    """A batch without rows: nothing to launch, gradients of zeros."""

    @staticmethod
    def forward(ctx, y, *others):
        ctx.save_for_backward(y, *others)
        return y.clone()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return tuple(torch.zeros_like(t) if need else None for t, need in zip(ctx.saved_tensors, ctx.needs_input_grad))


def _update(op, y, x, a, b, call, scaling, out, stream):
    """The checks that both forms share, and the call."""
    dev = x.device
    _refuse_tangents(op, y, x, a, b, scaling)
    if y.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"[mlx_kquant.{op}] y must be float16 or bfloat16 but is {y.dtype}.")
    if x.dtype != y.dtype:
        if x.dtype != torch.float32 or y.dtype != torch.bfloat16:   # what quantized_matmul makes of float32 rows
            raise ValueError(f"[mlx_kquant.{op}] x must be of y's dtype (or float32 beside bfloat16) but is {x.dtype}.")
        x = x.to(torch.bfloat16)
    if a.dtype != b.dtype or a.dtype not in (y.dtype, torch.float32):
        raise ValueError(f"[mlx_kquant.{op}] a and b must both be of y's dtype or float32 but are {a.dtype}, {b.dtype}.")
    r = a.shape[-2]
    if not 1 <= r <= MAX_RANK:
        raise ValueError(f"[mlx_kquant.{op}] the rank must be 1 to {MAX_RANK} but is {r}.")
    if a.shape[:-2] != b.shape[:-2] or b.shape[-1] != r or a.shape[-1] != x.shape[-1] or b.shape[-2] != y.shape[-1]:
        raise ValueError(f"[mlx_kquant.{op}] a {tuple(a.shape)} and b {tuple(b.shape)} do not fit x {tuple(x.shape)} and "
                         f"y {tuple(y.shape)}.")
    if not x.is_cuda or any(t.device != dev for t in (y, a, b)):
        raise RuntimeError(f"[mlx_kquant.{op}] y, x, a and b must live on one CUDA device; there is no CPU path.")
    call.n_adapters = a.shape[0]
    call.scale, call.scaling = 1.0, None
    if isinstance(scaling, torch.Tensor):
        if scaling.requires_grad:
            raise ValueError(f"[mlx_kquant.{op}] the scaling has no gradient: pass it detached.")
        if scaling.shape != (call.n_adapters,):
            raise ValueError(f"[mlx_kquant.{op}] scaling must be a number or of shape ({call.n_adapters},) but has "
                             f"{tuple(scaling.shape)}.")
        call.scaling = scaling.to(device=dev, dtype=torch.float32).contiguous()
    elif scaling is not None:
        call.scale = float(scaling)
    call.stream = stream
    grads = torch.is_grad_enabled() and (y.requires_grad or x.requires_grad or a.requires_grad or b.requires_grad)
    if out is not None:
        if grads:
            raise ValueError(f"[mlx_kquant.{op}] out= takes no part in gradients; leave it away.")
        if out.shape != y.shape or out.dtype != y.dtype or out.device != dev or not out.is_contiguous():
            raise ValueError(f"[mlx_kquant.{op}] out must be contiguous, of y's shape, dtype and device.")
        itself = out.data_ptr() == y.data_ptr() and y.is_contiguous()
        if any(_overlap(t, out) for t in ((x, a, b) if itself else (y, x, a, b))):
            raise ValueError(f"[mlx_kquant.{op}] out must not overlap x, a, b or, unless it is y, y.")
    if y.numel() == 0:
        return _Empty.apply(y, x, a, b) if grads else y.clone() if out is None else out
    if grads:
        if stream is not None:
            raise ValueError(f"[mlx_kquant.{op}] stream= takes no part in gradients; set the current stream instead.")
        return _Update.apply(call, y, x, a, b)
    rows = y.numel() // y.shape[-1]
    if out is None:
        out = torch.empty(y.shape, dtype=y.dtype, device=dev)
    call.forward(y, x, a, b, out, None, call.plan(rows, dev) if rows > DIRECT_ROWS else None)
    return out


def lora_update(y, x, a, b, adapter_ids=None, scaling=None, *, out=None, stream=None):
    """``y + scaling[g] * (x @ a[g].T) @ b[g].T``, row by row with the row's own adapter g.

    y [..., N]: what the shared projection gave, float16 or bfloat16; x [..., K]: its input, of the same dtype (float32 beside
    bfloat16 is rounded, as `quantized_matmul` does). a [G, r, K] and b [G, N, r]: the adapters, of y's dtype or float32 (without the
    first axis: one adapter); r <= 128. adapter_ids: int, of the shape of x's leading axes or of the first of them (one index
    for all rows below); outside [0, G): no adapter, the row stays y's. None: adapter 0 for every row. scaling: a number, or
    a tensor [G]; None: 1.

    Returns a tensor like y, or writes to `out`, which may be y but overlaps nothing else. Differentiable backwards in y, x, a and b (not
    with `out` or `stream`). The same call gives the same bits. A training step can be captured into a CUDA graph; as for every operator
    of torch, no eager autograd graph of the same leaves may be alive then."""
    if out is None and stream is None:
        done = front_update(y, x, a, b, adapter_ids, scaling, None)
        if done is not None:
            return done
    op = "lora_update"
    if a.dim() == 2 and b.dim() == 2:
        a, b = a.unsqueeze(0), b.unsqueeze(0)
    if a.dim() != 3 or b.dim() != 3:
        raise ValueError(f"[mlx_kquant.{op}] a must be [adapters, r, K] and b [adapters, N, r] but got shapes {tuple(a.shape)}, "
                         f"{tuple(b.shape)}.")
    if x.dim() < 1 or x.shape[:-1] != y.shape[:-1]:
        raise ValueError(f"[mlx_kquant.{op}] x {tuple(x.shape)} and y {tuple(y.shape)} must have the same rows.")
    call = _Call()
    call.shared, call.n_experts, call.experts, call.ids, call.slots = False, 1, None, None, 1
    if adapter_ids is not None:
        lead = adapter_ids.dim()
        if adapter_ids.shape != x.shape[:-1][:lead] or not _integers(adapter_ids):
            raise ValueError(f"[mlx_kquant.{op}] adapter_ids must be integers of x's leading axes {tuple(x.shape[:-1])} but got "
                             f"{adapter_ids.dtype} {tuple(adapter_ids.shape)}.")
        call.ids = _i32(adapter_ids, x.device)
        for d in x.shape[:-1][lead:]:
            call.slots *= d
        call.slots = max(1, call.slots)
    elif a.shape[0] != 1:
        raise ValueError(f"[mlx_kquant.{op}] {a.shape[0]} adapters need adapter_ids.")
    return _update(op, y, x, a, b, call, scaling, out, stream)


class _FrozenMatmul(torch.autograd.Function):
    """quantized_matmul with the gradient of its input; the wire bytes have none."""

    @staticmethod
    def forward(ctx, x, w, scales, kquant_type):
        ctx.kquant_type, ctx.dtype = kquant_type, x.dtype
        ctx.save_for_backward(w)
        return quantized_matmul(x.detach(), w, scales, kquant_type)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        w, = ctx.saved_tensors
        return quantized_matmul(dy, w, None, ctx.kquant_type, transpose=False).to(ctx.dtype), None, None, None


def quantized_matmul_lora(x, w, scales, kquant_type, a, b, adapter_ids=None, scaling=None, *, stream=None):
    """``quantized_matmul(x, w)`` with low-rank adapters on top (`lora_update`). The projection is rounded to the output dtype
    before the update is added, once more. Differentiable in x, a and b; the wire bytes stay as they are."""
    if torch.is_grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad):
        if stream is not None:
            raise ValueError("[mlx_kquant.quantized_matmul_lora] stream= takes no part in gradients; set the current stream instead.")
        y = _FrozenMatmul.apply(x, w, scales, kquant_type) if x.requires_grad else quantized_matmul(x, w, scales, kquant_type)
        return lora_update(y, x, a, b, adapter_ids, scaling)
    y = quantized_matmul(x, w, scales, kquant_type, stream=stream)
    return lora_update(y, x, a, b, adapter_ids, scaling, out=y, stream=stream)
