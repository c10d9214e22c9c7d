"""Linear layers of 8-bit blocks: e4m3 weights with one power-of-two scale for 128 x 128 of them (csrc/fp8_linear.hip).

    y = T( sum over blocks b of K of  sx[m, b] sw[n / 128, b]  sum over k in b of  xq[m, k] wq[n, k] )

The rows of x are quantised in the call, 128 columns at a time, each block under the least power of two that brings its
largest magnitude to at most 448.  Half the bytes of 16-bit weights for a decode step, twice their matrix rate for prompts.
The reference has no counterpart (its weights are 16-bit); its planned quantized serving is
docs/distributed_inference_plan.md:310.

`quantize_(model)` replaces the projections of every decoder layer; `Fp8Linear.from_parts` takes weights that were quantised
elsewhere.  For inference: a call whose input needs a gradient is refused.
"""

from __future__ import annotations

from contextlib import nullcontext

import torch
import torch.nn.functional as F
from torch import nn

from .. import _native
from . import kernels

BLOCK = 128
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TOP = 448.0  # e4m3's largest value, 1.75 * 2^8


def _scale_exponents(amax: torch.Tensor) -> torch.Tensor:
    """e8m0 codes of blocks of this largest magnitude (fp32): the least power of two with amax / 2^e <= 448; 255 for a block
    that is not finite."""
    e = ((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8
    return torch.where(torch.isfinite(amax), e.clamp(min=1), 255).to(torch.uint8)


def _powers(e: torch.Tensor) -> torch.Tensor:
    """2^(e - 127) of e8m0 codes, 255 NaN; of code 0, below float32's normal numbers, bit 22 alone."""
    bits = torch.where(e == 0, 1 << 22, e.int() << 23)
    return torch.where(e == 255, float("nan"), bits.view(torch.float32))


def _no_autocast(device_type: str):
    """A context in which a product keeps its operands' type, whatever autocast is on (meta tensors have none)."""
    return nullcontext() if device_type == "meta" else torch.autocast(device_type, enabled=False)


def quantize_blocks(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """weight [N, K] -> (e4m3 codes [N, K], e8m0 scales [ceil(N / 128), ceil(K / 128)])."""
    n, k = weight.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = F.pad(weight.float(), (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    e = _scale_exponents(w.abs().amax(dim=(1, 3)))
    codes = (w / _powers(e)[:, None, :, None]).to(E4M3).view(torch.uint8).view(nb * BLOCK, kb * BLOCK)
    return codes[:n, :k].contiguous().view(E4M3), e.view(E8M0)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] -> (e4m3 codes [M, 128 ceil(K / 128)], e8m0 scales [M, ceil(K / 128)]), as the kernels quantise it."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    b = F.pad(x.float(), (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    e = _scale_exponents(b.abs().amax(dim=2))
    return (b / _powers(e)[..., None]).to(E4M3).flatten(1), e.view(E8M0)


class Fp8Linear(nn.Module):
    """A bias-free linear layer of 8-bit blocks.  `weight` [out_features, in_features padded with zeros to a multiple of 128]
    e4m3, `weight_scale` [ceil(out / 128), ceil(in / 128)] e8m0; both sizes multiples of 16.  On a GPU it takes bfloat16 and
    float16 rows to the kernels; elsewhere, and under a compiler or another function mode, the same result comes from torch
    operations in float32.  torch.jit.trace and vmap, which have no rule for reading a number's bits, raise."""

    def __init__(self, in_features: int, out_features: int, device=None) -> None:
        super().__init__()
        if in_features <= 0 or out_features <= 0 or in_features % 16 or out_features % 16:
            raise ValueError(f"in_features and out_features must be positive multiples of 16, not {in_features}, {out_features}")
        self.in_features, self.out_features = in_features, out_features
        nb, kb = -(-out_features // BLOCK), -(-in_features // BLOCK)
        self.register_buffer("weight", torch.zeros((out_features, kb * BLOCK), dtype=torch.uint8, device=device).view(E4M3))
        self.register_buffer("weight_scale", torch.full((nb, kb), 127, dtype=torch.uint8, device=device).view(E8M0))

    @classmethod
    def from_parts(cls, weight: torch.Tensor, weight_scale: torch.Tensor) -> Fp8Linear:
        """From e4m3 codes [N, K] and e8m0 scales [ceil(N / 128), ceil(K / 128)]; codes of a K that is a multiple of 128 are kept,
        not copied."""
        if weight.dim() != 2 or weight.dtype != E4M3:
            raise ValueError("weight must be [N, K] float8_e4m3fn")
        n, k = weight.shape
        layer = cls(k, n, device="meta")
        if weight_scale.dtype != E8M0 or weight_scale.shape != layer.weight_scale.shape:
            raise ValueError(f"weight_scale must be {list(layer.weight_scale.shape)} float8_e8m0fnu")
        if weight_scale.device != weight.device:
            raise ValueError("weight and weight_scale must be on one device")
        if k % BLOCK:
            weight = F.pad(weight.view(torch.uint8), (0, -k % BLOCK)).view(E4M3)
        layer.weight, layer.weight_scale = weight.contiguous(), weight_scale.contiguous()
        return layer

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> Fp8Linear:
        if linear.bias is not None:
            raise ValueError("a layer of 8-bit blocks has no bias")
        with torch.no_grad():
            return cls.from_parts(*quantize_blocks(linear.weight.detach()))

    def _apply(self, fn, recurse=True):
        """Moves go through, casts leave codes and scales alone (Module.type casts bytes too: of that the device is kept)."""
        for name, dtype in (("weight", E4M3), ("weight_scale", E8M0)):
            held = self._buffers[name].view(torch.uint8)
            got = fn(held)
            self._buffers[name] = (got if got.dtype == torch.uint8 else held.to(got.device)).view(dtype)
        return self

    def dequantized(self) -> torch.Tensor:
        """The weights' values, float32 [out_features, in_features]."""
        s = _powers(self.weight_scale.view(torch.uint8)).repeat_interleave(BLOCK, 0)[:self.out_features]
        return (self.weight.float() * s.repeat_interleave(BLOCK, 1))[:, :self.in_features]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"x must have {self.in_features} columns, not {x.shape[-1]}")
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError("Fp8Linear is for inference: its rounding of x has no gradient (call it under no_grad)")
        if kernels.usable(x, grad_ok=True):
            y = self._kernel(x)
            if y is not None:
                return y
        elif not torch.compiler.is_compiling() and x.is_cuda and not _native.available():
            _native.lib()  # raises: a GPU without the library is an error
        codes, e = quantize_rows(x.reshape(-1, self.in_features))
        rows = (codes.float().unflatten(1, (-1, BLOCK)) * _powers(e.view(torch.uint8))[..., None]).flatten(1)
        with _no_autocast(x.device.type):
            y = rows[:, :self.in_features] @ self.dequantized().t()
        return y.to(x.dtype).view(*x.shape[:-1], self.out_features)

    def _kernel(self, x: torch.Tensor) -> torch.Tensor | None:
        """The library's product, or None for operands that it does not take."""
        k, n, device = self.in_features, self.out_features, x.device
        w, s = self._buffers["weight"], self._buffers["weight_scale"]
        m = x.numel() // k
        if not (w.device == device == s.device and w.is_contiguous() and s.is_contiguous() and w.data_ptr() % 16 == 0
                and s.data_ptr() % 4 == 0 and k <= 1 << 23 and n < 1 << 28 and m * w.shape[1] <= kernels.MAX_GROUPS * 4096):
            return None
        if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) % 8 == 0 and x.data_ptr() % 16 == 0:
            rows, stride = x, x.stride(0)
        else:
            rows, stride = x.contiguous(), k
            if rows.data_ptr() % 16:
                rows = rows.clone()
        out = x.new_empty((*x.shape[:-1], n))
        if m == 0:
            return out
        lib = _native.lib()
        size = lib.fn("mllm_fp8_linear_workspace_bytes")(m, n, k, 0)
        work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        lib.launch(device, "mllm_fp8_linear", rows.data_ptr(), stride, m, k, w.data_ptr(), s.data_ptr(), n,
                   _native.dtype_code(x.dtype), None if work is None else work.data_ptr(), size, out.data_ptr())
        return out

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}"


@torch.no_grad()
def quantize_(model: nn.Module) -> nn.Module:
    """Replaces the projections of every decoder layer of `model` (LlamaForCausalLM) by layers of 8-bit blocks, in place.  The
    embedding and lm_head keep their weights.  A projection that does more than nn.Linear (a forward of its own, hooks) is
    refused: the layer in its place would not do it."""
    places = [(owner, name) for layer in model.model.layers
              for owner, names in ((layer.self_attn, ("q_proj", "k_proj", "v_proj", "o_proj")),
                                   (layer.mlp, ("gate_proj", "up_proj", "down_proj")))
              for name in names if isinstance(getattr(owner, name), nn.Linear)]
    for owner, name in places:  # all or none
        linear = getattr(owner, name)
        if linear.bias is not None or linear.in_features % 16 or linear.out_features % 16:
            raise ValueError(f"{name} must have no bias and sizes that are multiples of 16, not {linear}")
        held = linear.__dict__
        if type(linear).forward is not nn.Linear.forward or "forward" in held or any(
                held[hooks] for hooks in ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")):
            raise ValueError(f"{name} must be a linear layer without a forward or hooks of its own, not {linear}")
    for owner, name in places:
        setattr(owner, name, Fp8Linear.from_linear(getattr(owner, name)))
    return model
