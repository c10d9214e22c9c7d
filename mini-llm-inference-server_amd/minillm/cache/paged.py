"""Paged KV pool (reference src/minillm/cache/paged.py:21-69).

Per layer, separate K and V tensors [num_blocks, block_size, Hkv, Dh] (NHD: token-major inside a
block), zero-initialised and allocated once; a block id names the same slot range in every layer.
Token p of a sequence lives at block_ids[p // block_size], offset p % block_size.  On an MI355X the
pool is sized from the 288 GB of HBM: one 16-token block of Llama-3.1-8B is 64 KB per layer, 2 MB
across its 32 layers.

A pool of dtype torch.float8_e4m3fn (the reference's planned fp8 KV cache, M9b in
docs/distributed_inference_plan.md:310) stores e4m3fn(x / scale) with one scale per tensor: `k_scale[l]`
and `v_scale[l]` for layer l, which the model passes to the backend with the layer's pools.  One block of
Llama-3.1-8B is then 32 KB per layer, so the same HBM holds twice the tokens.

A pool of dtype torch.float4_e2m1fn_x2 stores 4-bit codes with a power-of-two scale for 32 dims of a token and head: the
pools are [num_blocks, block_size, Hkv, Dh / 2] (two codes to a byte), `k_scale[l]` [num_blocks, block_size, Dh / 32, Hkv]
and `v_scale[l]` [num_blocks, Hkv, Dh / 32, block_size] torch.float8_e8m0fnu tensors (include/minillm_hip.h has the
format).  One block of Llama-3.1-8B is 17 KB per layer, so the same HBM holds 3.76 times the tokens of 16 bits.

`PagedStep` is the pool as one forward pass sees it: the pool plus that step's metadata.
"""

from __future__ import annotations

import torch

from .. import _native

BLOCK_SIZE = 16
FP4 = torch.float4_e2m1fn_x2
FP4_BLOCK = 32  # dims per scale of a 4-bit pool


class PagedKVCache:
    def __init__(self, config, num_blocks: int, device: torch.device | str, dtype: torch.dtype,
                 block_size: int = BLOCK_SIZE, k_scale: float = 1.0, v_scale: float = 1.0) -> None:
        hkv, dh = config.num_key_value_heads, config.head_dim
        self.fp4 = dtype == FP4
        if self.fp4 and dh % (2 * FP4_BLOCK):
            raise ValueError(f"a 4-bit pool needs a head_dim that is a multiple of {2 * FP4_BLOCK}, not {dh}")
        self.head_dim = dh
        shape = (num_blocks, block_size, hkv, dh // 2 if self.fp4 else dh)
        zeros = torch.uint8 if self.fp4 else dtype  # torch fills no 4-bit tensor on a GPU
        self.k = [torch.zeros(shape, device=device, dtype=zeros).view(dtype) for _ in range(config.num_hidden_layers)]
        self.v = [torch.zeros(shape, device=device, dtype=zeros).view(dtype) for _ in range(config.num_hidden_layers)]
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.quantized = dtype == torch.float8_e4m3fn
        if not self.quantized and (k_scale != 1.0 or v_scale != 1.0):
            raise ValueError("k_scale / v_scale apply to fp8 pools only")
        self.k_scale: list = [float(k_scale)] * config.num_hidden_layers
        self.v_scale: list = [float(v_scale)] * config.num_hidden_layers
        if self.fp4:
            blocks = dh // FP4_BLOCK
            for scales, of in ((self.k_scale, (num_blocks, block_size, blocks, hkv)),
                               (self.v_scale, (num_blocks, hkv, blocks, block_size))):
                scales[:] = [torch.zeros(of, device=device, dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in scales]

    def scales(self, layer: int) -> dict:
        """Keyword arguments of the backend call for `layer`: its scales for an fp8 or 4-bit pool, none otherwise."""
        return {"k_scale": self.k_scale[layer], "v_scale": self.v_scale[layer]} if self.quantized or self.fp4 else {}

    def read(self, layer: int, slots: torch.Tensor, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values of K and V at `slots` [n] (int64, on the pool's device; as a step's slot_mapping names them), both
        [n, Hkv, Dh] of `dtype`: by default the pool's own, bfloat16 for fp8 and 4-bit pools.  A 4-bit pool is read with the
        16-bit type it was written with.  A slot outside the pool reads as zeros."""
        k, v = self.k[layer], self.v[layer]
        device = k.device
        if slots.dim() != 1 or slots.dtype != torch.int64 or slots.device != device:
            raise ValueError("slots must be one row of int64 on the pool's device")
        dtype = dtype or (torch.bfloat16 if self.quantized or self.fp4 else k.dtype)
        if not self.fp4:
            got, outside = [], (slots < 0) | (slots >= k.shape[0] * k.shape[1])
            slots = slots.masked_fill(outside, 0)
            for pool, scale in ((k, self.k_scale[layer]), (v, self.v_scale[layer])):
                raw = pool.view(torch.uint8) if self.quantized else pool
                rows = raw.flatten(0, 1).index_select(0, slots)
                rows = rows.view(pool.dtype).float() * scale if self.quantized else rows
                got.append(rows.masked_fill(outside[:, None, None], 0).to(dtype))
            return got[0], got[1]
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("a 4-bit pool is read as bfloat16 or float16")
        if device.type != "cuda":
            raise RuntimeError(f"reading a 4-bit pool needs a GPU device, got {device}")
        nb, bs, hkv, half = k.shape
        slots = slots.contiguous()
        n = slots.numel()
        to_k, to_v = torch.empty((2, n, hkv, 2 * half), dtype=dtype, device=device).unbind()
        _native.lib().launch(device, "mllm_kv_read_fp4", k.data_ptr(), v.data_ptr(), self.k_scale[layer].data_ptr(),
                             self.v_scale[layer].data_ptr(), nb, bs, hkv, 2 * half, slots.data_ptr(), n,
                             _native.dtype_code(dtype), to_k.data_ptr(), to_v.data_ptr())
        return to_k, to_v

    @staticmethod
    def bytes_per_block(config, dtype: torch.dtype, block_size: int = BLOCK_SIZE) -> int:
        """K and V, every layer: 2 x layers x block_size x KV heads x head_dim x bytes per element (4-bit pools: half a
        byte, and a scale byte for 32 dims)."""
        if dtype == FP4:
            row = config.head_dim // 2 + config.head_dim // FP4_BLOCK
            return 2 * config.num_hidden_layers * block_size * config.num_key_value_heads * row
        elem = torch.tensor([], dtype=dtype).element_size()
        return 2 * config.num_hidden_layers * block_size * config.num_key_value_heads * config.head_dim * elem

    @classmethod
    def blocks_for_bytes(cls, config, dtype: torch.dtype, num_bytes: int, block_size: int = BLOCK_SIZE) -> int:
        return num_bytes // cls.bytes_per_block(config, dtype, block_size)

    def step(self, meta) -> PagedStep:
        return PagedStep(self, meta)


class PagedStep:
    """What a model's forward pass calls on its KV cache for one ragged step.  The backend's `forward`
    reads and writes the pool itself, so there is nothing to mark or advance."""

    ragged = True

    def __init__(self, cache: PagedKVCache, meta) -> None:
        self.cache, self.meta = cache, meta

    def positions(self, input_ids: torch.Tensor, attention_mask: torch.Tensor | None = None) -> torch.Tensor:
        return self.meta.positions[None, :]

    def mark(self, attention_mask: torch.Tensor | None, num_tokens: int) -> None:
        if attention_mask is not None:
            raise ValueError("a ragged step has no padding, so no attention mask")

    def key_valid(self, num_new: int) -> None:
        return None

    def advance(self, num_tokens: int) -> None:
        pass
