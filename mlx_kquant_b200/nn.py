"""torch modules over GGUF wire bytes, the counterparts of the reference's module layer
(mlx_kquant/nn.py:50-268): `KQuantEmbedding`, `KQuantLinear`, `KQuantSwitchLinear`, and low-rank adapters on the last two:
`KQuantLoRALinear`, `KQuantLoRASwitchLinear`.

Each keeps `weight` as a uint8 buffer of wire bytes (never a float copy) and a one-byte `scales`
placeholder, so that a state dict has the reference's keys and shapes, and calls the `kq.*` ops.
"""
from __future__ import annotations

import os

import torch

from . import _lib
from . import ops as kq
from .lora import _FrozenMatmul, _i32, lora_update
from .moe import gather_lora_update


def bytes_per_row(codec: str, dims: int) -> int:
    """Wire bytes of one row of `dims` weights (mlx_kquant/codec_geometry.py)."""
    wpb, bpb, _, _ = kq.codec_geometry(codec)
    if dims % wpb != 0:
        raise ValueError(f"[mlx_kquant] {dims} weights per row is not a whole number of {wpb}-weight {codec} blocks.")
    return dims // wpb * bpb


def _dims(layer) -> int:
    """Weights in a row of a layer's wire bytes."""
    wpb, bpb, _, _ = kq.codec_geometry(layer.kquant_type)
    return layer.weight.shape[-1] // bpb * wpb


class _KQuantBase(torch.nn.Module):
    def _init_codec(self, codec: str) -> None:
        wpb, _, bits, _ = kq.codec_geometry(codec)
        self.mode = "kquant"
        self.group_size = wpb
        self.bits = bits
        self.kquant_type = codec
        self.register_buffer("scales", torch.zeros(1, dtype=torch.uint8))


class KQuantEmbedding(_KQuantBase):
    """Embedding table in wire bytes (mlx_kquant/nn.py:50-96): a lookup gathers the tokens' wire rows and
    dequantizes only those; `as_linear` is the tied output projection."""

    def __init__(self, num_embeddings: int, dims: int, codec: str, out_dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self._init_codec(codec)
        self.num_embeddings, self.dims, self.out_dtype = num_embeddings, dims, out_dtype
        self.register_buffer("weight", torch.zeros((num_embeddings, bytes_per_row(codec, dims)), dtype=torch.uint8))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        rows = self.weight[x.to(self.weight.device).reshape(-1)]
        deq = kq.dequantize(rows, self.scales, self.kquant_type, self.out_dtype)
        return deq.reshape(*x.shape, self.dims)

    def as_linear(self, x: torch.Tensor) -> torch.Tensor:
        return kq.quantized_matmul(x, self.weight, self.scales, self.kquant_type, transpose=True)

    def extra_repr(self) -> str:
        return f"{self.num_embeddings}, {self.dims}, kquant_type={self.kquant_type}"


class KQuantLinear(_KQuantBase):
    """Linear layer in wire bytes (mlx_kquant/nn.py:99-158): weight [out_dims, bytes_per_row]."""

    def __init__(self, in_dims: int, out_dims: int, bias: bool, codec: str):
        super().__init__()
        self._init_codec(codec)
        self.register_buffer("weight", torch.zeros((out_dims, bytes_per_row(codec, in_dims)), dtype=torch.uint8))
        if bias:
            self.register_buffer("bias", torch.zeros(out_dims))
        else:
            self.bias = None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        # decode (one row) with a bias: the add is fused into the q8_0 decode kernel, as the reference does
        # (mlx_kquant/nn.py:129-146); KQ_DISABLE_QMV_BIAS=1 forces the unfused path, read live
        if (self.bias is not None and self.kquant_type == "q8_0" and x.numel() // x.shape[-1] == 1
                and os.environ.get("KQ_DISABLE_QMV_BIAS") != "1"):
            return kq.quantized_matmul_qmv_bias(x, self.weight, self.scales, self.bias, self.kquant_type)
        y = kq.quantized_matmul(x, self.weight, self.scales, self.kquant_type, transpose=True)
        if self.bias is not None:
            y = y + self.bias.to(y.dtype)
        return y

    def extra_repr(self) -> str:
        out_dims, bpr = self.weight.shape
        return f"output_dims={out_dims}, bytes_per_row={bpr}, kquant_type={self.kquant_type}"


class KQuantSwitchLinear(_KQuantBase):
    """Expert stack in wire bytes (mlx_kquant/nn.py:161-268): weight [n_experts, out_dims, bytes_per_row];
    `forward(x, indices, sorted_indices)` is `gather_qmm` over the stack. Prefill-shaped sorted calls
    (x [B, 1, K], indices [B] ascending, B >= KQ_SWITCH_GEMM_MIN_ROWS, default 512) take the segment product
    with a device-built tile map, which needs no host read of the routing."""

    def __init__(self, num_experts: int, output_dims: int, input_dims: int, bias: bool, codec: str):
        super().__init__()
        self._init_codec(codec)
        self.register_buffer("weight", torch.zeros((num_experts, output_dims, bytes_per_row(codec, input_dims)),
                                                   dtype=torch.uint8))
        if bias:
            self.register_buffer("bias", torch.zeros((num_experts, output_dims)))
        else:
            self.bias = None

    def forward(self, x: torch.Tensor, indices: torch.Tensor, sorted_indices: bool = False) -> torch.Tensor:
        if (sorted_indices and indices.dim() == 1 and x.dim() == 3 and x.shape[0] == indices.numel()
                and x.shape[1] == 1):
            min_rows = int(os.environ.get("KQ_SWITCH_GEMM_MIN_ROWS", "512"))
            if min_rows > 0 and indices.numel() >= min_rows:
                y = self._sorted_expert_gemm(x, indices)
                return self._add_bias(y, indices)
        y = kq.gather_qmm(x, self.weight, self.scales, self.kquant_type, rhs_indices=indices, transpose=True,
                          sorted_indices=sorted_indices)
        return self._add_bias(y, indices)

    def _add_bias(self, y: torch.Tensor, indices: torch.Tensor) -> torch.Tensor:
        if self.bias is None:
            return y
        return y + self.bias[indices.to(self.bias.device).long()].unsqueeze(-2).to(y.dtype)

    def _sorted_expert_gemm(self, x: torch.Tensor, indices: torch.Tensor) -> torch.Tensor:
        xf = x.reshape(indices.numel(), -1)
        idx = indices.to(self.weight.device)
        maps = kq.expert_tile_map(idx.to(torch.int32), self.weight.shape[0])
        return kq.gather_qmm_seg(xf, self.weight, self.scales, self.kquant_type, *maps)[:, None, :]

    def extra_repr(self) -> str:
        n, m, b = self.weight.shape
        return f"num_experts={n}, output_dims={m}, bytes_per_row={b}, kquant_type={self.kquant_type}"


class KQuantMultiLinear(_KQuantBase):
    """Per-head batched linear in wire bytes (mlx_kquant/nn.py:271-352), the absorbed-attention up-projections of
    the deepseek_v3 family: weight [num_heads, out_dims, bytes_per_row], dispatched through `gather_qmm` with the
    head as the expert index. `forward(x, transpose)`: x is [B, Hx, L, D] with Hx = num_heads (per-head
    activations) or 1 (one activation shared by all heads); `transpose=True` computes x[..., h, :, :] @ W[h].T,
    `transpose=False` computes x @ W[h] (contraction over the axis that is not quantized)."""

    def __init__(self, input_dims: int, output_dims: int, num_heads: int, codec: str):
        super().__init__()
        self._init_codec(codec)
        self.num_heads = num_heads
        self.register_buffer("weight", torch.zeros((num_heads, output_dims, bytes_per_row(codec, input_dims)),
                                                   dtype=torch.uint8))
        self._gather_idx = None

    def forward(self, x: torch.Tensor, transpose: bool = True) -> torch.Tensor:
        nh = self.num_heads
        B, Hx = x.shape[0], x.shape[1]
        dev = self.weight.device
        cached = self._gather_idx
        if cached is not None and cached[0] == (B, Hx, dev):
            lhs, rhs = cached[1], cached[2]
        else:
            rhs = torch.arange(nh, dtype=torch.int32, device=dev).reshape(1, nh).expand(B, nh).contiguous()
            if Hx == nh:
                lhs = torch.arange(B * nh, dtype=torch.int32, device=dev).reshape(B, nh)
            elif Hx == 1:
                lhs = torch.arange(B, dtype=torch.int32, device=dev).reshape(B, 1).expand(B, nh).contiguous()
            else:
                raise ValueError(f"KQuantMultiLinear: head axis {Hx} is neither 1 nor num_heads={nh} "
                                 f"(x.shape={tuple(x.shape)})")
            self._gather_idx = ((B, Hx, dev), lhs, rhs)
        return kq.gather_qmm(x, self.weight, self.scales, self.kquant_type, lhs_indices=lhs, rhs_indices=rhs,
                             transpose=transpose)

    def extra_repr(self) -> str:
        nh, out_dims, bpr = self.weight.shape
        return f"num_heads={nh}, output_dims={out_dims}, bytes_per_row={bpr}, kquant_type={self.kquant_type}"


class KQuantLoRALinear(torch.nn.Module):
    """Low-rank adapters on a `KQuantLinear` (the counterpart of an adapter layer over frozen quantized weights): `lora_a`
    [n_adapters, rank, in_dims] and `lora_b` [n_adapters, out_dims, rank], zero at first, are its parameters, `scaling` a factor
    for each adapter. `forward(x, adapter_ids)` gives every row the adapter of its request (`lora_update`); a training step reaches x and
    the parameters, the wire bytes stay as they are."""

    def __init__(self, base: KQuantLinear, rank: int, n_adapters: int = 1, scaling: float = 1.0, dtype: torch.dtype = torch.float32):
        super().__init__()
        out_dims, in_dims = base.weight.shape[0], _dims(base)
        self.base = base
        dev = base.weight.device
        self.lora_a = torch.nn.Parameter((torch.rand(n_adapters, rank, in_dims, device=dev) * 2 - 1).mul_(in_dims ** -0.5).to(dtype))
        self.lora_b = torch.nn.Parameter(torch.zeros(n_adapters, out_dims, rank, dtype=dtype, device=dev))
        self.register_buffer("scaling", torch.full((n_adapters,), float(scaling), device=dev))

    def forward(self, x: torch.Tensor, adapter_ids: torch.Tensor | None = None) -> torch.Tensor:
        base = self.base
        if torch.is_grad_enabled() and x.requires_grad:
            y = _FrozenMatmul.apply(x, base.weight, base.scales, base.kquant_type)
            if base.bias is not None:
                y = y + base.bias.to(y.dtype)
        else:
            y = base(x)
        return lora_update(y, x, self.lora_a, self.lora_b, adapter_ids, self.scaling)

    def extra_repr(self) -> str:
        n, r, _ = self.lora_a.shape
        return f"rank={r}, n_adapters={n}"


def _clear(y: torch.Tensor, indices: torch.Tensor, n_experts: int) -> torch.Tensor:
    """y's rows of indices (int32) outside the stack, which the products leave unwritten, become zero."""
    with kq._on_device(y.device):
        kq.check(_lib.lib().kq_clear_rows(y.data_ptr(), indices.numel(), y.shape[-1], indices.data_ptr(), n_experts, kq._stream_ptr(None, y.device)))
    return y


def _routed(base: KQuantSwitchLinear, x: torch.Tensor, indices: torch.Tensor, sorted_indices: bool) -> torch.Tensor:
    """The stack's products with rows of zeros where an index (int32) lies outside of it."""
    E, near = base.weight.shape[0], indices
    if base.bias is not None or sorted_indices:   # a bias is looked up for all, and the segments of sorted rows have no room for others
        near = indices.clamp(0, E - 1)
    return _clear(base(x, near, sorted_indices), indices, E)


class _FrozenGather(torch.autograd.Function):
    """_routed with the gradient of its rows; the wire bytes have none."""

    @staticmethod
    def forward(ctx, x, base, indices):
        ctx.kquant_type, ctx.x_shape, ctx.dtype = base.kquant_type, x.shape, x.dtype
        ctx.save_for_backward(base.weight, indices)
        return _routed(base, x.detach(), indices, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        w, indices = ctx.saved_tensors
        dx = _clear(kq.gather_qmm(dy, w, None, ctx.kquant_type, rhs_indices=indices, transpose=False), indices, w.shape[0])
        return dx.float().sum_to_size(ctx.x_shape).to(ctx.dtype), None, None


class KQuantLoRASwitchLinear(torch.nn.Module):
    """Low-rank adapters on a `KQuantSwitchLinear`: a pair of matrices for every adapter and expert, `lora_a` [n_adapters, n_experts,
    rank, in_dims], `lora_b` [n_adapters, n_experts, out_dims, rank]. `forward(x, indices, adapter_ids, sorted_indices)` takes what the
    base takes for routed rows: indices [T, R] with x [T, 1, 1, K] (one row per token) or [T, R, 1, K] and adapter_ids [T], or
    indices [B] with x [B, 1, K] and adapter_ids [B] (`moe.gather_lora_update`). Rows of an index outside the stack, as the router's
    -1, are zero, without bias."""

    def __init__(self, base: KQuantSwitchLinear, rank: int, n_adapters: int = 1, scaling: float = 1.0,
                 dtype: torch.dtype = torch.float32):
        super().__init__()
        (n_experts, out_dims, _), in_dims = base.weight.shape, _dims(base)
        self.base = base
        dev = base.weight.device
        self.lora_a = torch.nn.Parameter(
            (torch.rand(n_adapters, n_experts, rank, in_dims, device=dev) * 2 - 1).mul_(in_dims ** -0.5).to(dtype))
        self.lora_b = torch.nn.Parameter(torch.zeros(n_adapters, n_experts, out_dims, rank, dtype=dtype, device=dev))
        self.register_buffer("scaling", torch.full((n_adapters,), float(scaling), device=dev))

    def forward(self, x: torch.Tensor, indices: torch.Tensor, adapter_ids: torch.Tensor | None = None,
                sorted_indices: bool = False) -> torch.Tensor:
        base, K = self.base, x.shape[-1]
        flat = indices.dim() == 1 and x.dim() == 3 and x.shape[:2] == (indices.shape[0], 1)
        if not flat and not (indices.dim() == 2 and x.dim() == 4 and x.shape[0] == indices.shape[0] and x.shape[2] == 1
                             and x.shape[1] in (1, indices.shape[1])):
            raise ValueError(f"KQuantLoRASwitchLinear: x must be [T, 1, 1, K] or [T, R, 1, K] with indices [T, R], or [B, 1, K] with "
                             f"indices [B], but x is {tuple(x.shape)} and indices {tuple(indices.shape)}.")
        if not x.is_cuda:
            raise RuntimeError("KQuantLoRASwitchLinear: x must live on a CUDA device; there is no CPU path.")
        indices = _i32(indices, base.weight.device)
        if torch.is_grad_enabled() and x.requires_grad:
            y = _FrozenGather.apply(x, base, indices)
        else:
            y = _routed(base, x, indices, sorted_indices)
        slots = indices.reshape(-1, 1) if flat else indices
        T, R = slots.shape
        rows = x.reshape(T, R, K) if flat or x.shape[1] == R else x.reshape(T, K)
        return gather_lora_update(y.reshape(T, R, y.shape[-1]), rows, self.lora_a, self.lora_b, slots, adapter_ids, self.scaling).reshape(y.shape)

    def extra_repr(self) -> str:
        n, e, r, _ = self.lora_a.shape
        return f"rank={r}, n_adapters={n}, n_experts={e}"
