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

With `block_scales`, a pool of dtype torch.float8_e4m3fn has a power-of-two scale for each page and head instead of one per
tensor: `k_scale[l]` and `v_scale[l]` are torch.float8_e8m0fnu tensors [num_blocks, Hkv].  They follow the tokens that come
into a page (include/minillm_hip.h has the rule), so there is nothing to calibrate, and nothing saturates but magnitudes
above 57,344 in fp16 (2.98e38 in bf16); one byte for 16 tokens of a head.

`PagedStep` is the pool as one forward pass sees it: the pool plus that step's metadata.
"""

from __future__ import annotations

import struct
from array import array

import numpy as np
import torch

from .. import _native
from ..attention.hip_backend import check_scales

BLOCK_SIZE = 16
FP4 = torch.float4_e2m1fn_x2
FP4_BLOCK = 32  # dims per scale of a 4-bit pool
MAX_PAGE_BYTES = (1 << 23) - 1  # of one tensor, that mllm_copy_pages takes
FP8 = torch.float8_e4m3fn
_data_ptr, _nbytes, _is_contiguous = torch.Tensor.data_ptr, torch.Tensor.nbytes.__get__, torch.Tensor.is_contiguous


class PagedKVCache:
    def __init__(self, config, num_blocks: int, device: torch.device | str, dtype: torch.dtype,
                 block_size: int = BLOCK_SIZE, k_scale: float = 1.0, v_scale: float = 1.0,
                 block_scales: bool = False) -> None:
        hkv, dh = config.num_key_value_heads, config.head_dim
        self.fp4 = dtype == FP4
        if self.fp4 and dh % (2 * FP4_BLOCK):
            raise ValueError(f"a 4-bit pool needs a head_dim that is a multiple of {2 * FP4_BLOCK}, not {dh}")
        self.block_scales = bool(block_scales)
        if self.block_scales:
            if dtype != FP8:
                raise ValueError("block_scales is for pools of float8_e4m3fn (a 4-bit pool always has them)")
            if dh != 128 or block_size not in (16, 32, 64):
                raise ValueError(f"a pool with block scales needs a head_dim of 128 and blocks of 16, 32 or 64 tokens, not "
                                 f"{dh} and {block_size}")
        self.head_dim = dh
        shape = (num_blocks, block_size, hkv, dh // 2 if self.fp4 else dh)
        zeros = torch.uint8 if self.fp4 else dtype  # torch fills no 4-bit tensor on a GPU
        self.k = [torch.zeros(shape, device=device, dtype=zeros).view(dtype) for _ in range(config.num_hidden_layers)]
        self.v = [torch.zeros(shape, device=device, dtype=zeros).view(dtype) for _ in range(config.num_hidden_layers)]
        self.num_blocks = num_blocks
        self.block_size = block_size
        self._pages: tuple | None = None  # _page_tensors
        self.quantized = dtype == FP8
        if (not self.quantized or self.block_scales) and (k_scale != 1.0 or v_scale != 1.0):
            raise ValueError("k_scale / v_scale apply to fp8 pools only, and not with block_scales")
        self.k_scale: list = [float(k_scale)] * config.num_hidden_layers
        self.v_scale: list = [float(v_scale)] * config.num_hidden_layers
        if self.fp4:
            blocks = dh // FP4_BLOCK
            for scales, of in ((self.k_scale, (num_blocks, block_size, blocks, hkv)),
                               (self.v_scale, (num_blocks, hkv, blocks, block_size))):
                scales[:] = [torch.zeros(of, device=device, dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in scales]
        elif self.block_scales:
            for scales in (self.k_scale, self.v_scale):
                scales[:] = [_page_scales(num_blocks, hkv, device) for _ in scales]

    def scales(self, layer: int) -> dict:
        """Keyword arguments of the backend call for `layer`: its scales for an fp8 or 4-bit pool, none otherwise."""
        return {"k_scale": self.k_scale[layer], "v_scale": self.v_scale[layer]} if self.quantized or self.fp4 else {}

    def read(self, layer: int, slots: torch.Tensor, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values of K and V at `slots` [n] (int64, on the pool's device; as a step's slot_mapping names them), both
        [n, Hkv, Dh] of `dtype`: by default the pool's own, bfloat16 for fp8 and 4-bit pools.  A pool with block scales is read
        with the 16-bit type it was written with.  A slot outside the pool reads as zeros."""
        k, v = self.k[layer], self.v[layer]
        device = k.device
        if slots.dim() != 1 or slots.dtype != torch.int64 or slots.device != device:
            raise ValueError("slots must be one row of int64 on the pool's device")
        dtype = dtype or (torch.bfloat16 if self.quantized or self.fp4 else k.dtype)
        if not (self.fp4 or self.block_scales):
            got, outside = [], (slots < 0) | (slots >= k.shape[0] * k.shape[1])
            slots = slots.masked_fill(outside, 0)
            for pool, scale in ((k, self.k_scale[layer]), (v, self.v_scale[layer])):
                raw = pool.view(torch.uint8) if self.quantized else pool
                rows = raw.flatten(0, 1).index_select(0, slots)
                rows = rows.view(pool.dtype).float() * scale if self.quantized else rows
                got.append(rows.masked_fill(outside[:, None, None], 0).to(dtype))
            return got[0], got[1]
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"{'a 4-bit pool' if self.fp4 else 'a pool with block scales'} is read as bfloat16 or float16")
        if v.shape != k.shape or v.dtype != k.dtype or not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("the pools must be alike and contiguous")
        check_scales(k, self.k_scale[layer], self.v_scale[layer])
        if device.type != "cuda":
            raise RuntimeError(f"reading {'a 4-bit pool' if self.fp4 else 'a pool with block scales'} needs a GPU device, got "
                               f"{device}")
        nb, bs, hkv, _ = k.shape
        dh = self.head_dim
        slots = slots.contiguous()
        n = slots.numel()
        to_k, to_v = torch.empty((2, n, hkv, dh), dtype=dtype, device=device).unbind()
        _native.lib().launch(device, "mllm_kv_read_fp4" if self.fp4 else "mllm_kv_read_fp8_blocks", k.data_ptr(),
                             v.data_ptr(), self.k_scale[layer].data_ptr(), self.v_scale[layer].data_ptr(), nb, bs, hkv, dh,
                             slots.data_ptr(), n, _native.dtype_code(dtype), to_k.data_ptr(), to_v.data_ptr())
        return to_k, to_v

    def copy_blocks(self, src, dst) -> None:
        """Block dst[i] becomes a copy of block src[i], in every layer's K, V and scales: one call on the current stream of the
        pool's device.  `src` and `dst` are sequences of block ids on the host, of one length.  A block written twice, or read
        and written, is refused (ValueError), as is one outside the pool; nothing is copied then.  On a GPU a block of one tensor
        may be of up to 8 MiB - 1."""
        src, dst = _block_ids(src), _block_ids(dst)
        n = len(src)
        if n != len(dst):
            raise ValueError(f"{n} blocks to copy from and {len(dst)} to copy to")
        if not n:
            return
        device = self.k[0].device
        if device.type != "cuda":
            self._copy_on_host(np.asarray(src), np.asarray(dst))
            return
        _native.lib().launch(device, "mllm_copy_pages", *self._page_tensors(), self.num_blocks, src.tobytes(), dst.tobytes(), n)

    def check_pages(self) -> None:
        """ValueError unless `copy_blocks` can take the pools and their scales as they are."""
        self._page_tensors()

    def _copy_on_host(self, src: np.ndarray, dst: np.ndarray) -> None:
        """`copy_blocks` of a pool that is not on a GPU, in torch operations, under the same rules."""
        for b in np.concatenate([src, dst]):
            if not 0 <= b < self.num_blocks:
                raise ValueError(f"block {b} is outside the pool")
        if np.unique(dst).size != dst.size:
            raise ValueError("a block is written twice")
        if np.intersect1d(src, dst).size:
            raise ValueError("a block is read and written")
        src, dst = torch.from_numpy(src), torch.from_numpy(dst)
        self._page_tensors()  # its checks
        for t in (*self.k, *self.v, *((*self.k_scale, *self.v_scale) if self.fp4 or self.block_scales else ())):
            raw = t.view(torch.uint8)
            raw[dst] = raw[src]

    def _page_tensors(self):
        """The addresses of every tensor that holds pages, and their bytes per page, as arrays mllm_copy_pages reads, and their
        number: checked and packed once, and again when one of them lies elsewhere or spans other bytes (an entry replaced, storage
        swapped, a view of the same memory).  Pages are bytes here, so these say all that the copies go by.  Asking 64 tensors takes
        the host 8 us, 3 of it their addresses alone."""
        tensors = [*self.k, *self.v]
        if self.fp4 or self.block_scales:
            tensors += self.k_scale
            tensors += self.v_scale
        addresses = list(map(_data_ptr, tensors))
        span = (self.num_blocks, list(map(_nbytes, tensors)))
        held = self._pages
        if held is not None and addresses == held[0] and span == held[1] and all(map(_is_contiguous, tensors)):
            return held[2:]
        for t in tensors:
            if t.shape[0] != self.num_blocks or not t.is_contiguous() or t.device != self.k[0].device:
                raise ValueError(f"the pools and their scales must be contiguous, of {self.num_blocks} blocks, on one device")
        nbytes = [n // max(1, self.num_blocks) for n in span[1]]
        if tensors[0].is_cuda and max(nbytes) > MAX_PAGE_BYTES:
            raise ValueError(f"pages of {max(nbytes)} bytes are too large to copy: at most {MAX_PAGE_BYTES}")
        self._pages = (addresses, span, struct.pack(f"{len(tensors)}Q", *addresses), struct.pack(f"{len(tensors)}q", *nbytes),
                       len(tensors))
        return self._pages[2:]

    @staticmethod
    def bytes_per_block(config, dtype: torch.dtype, block_size: int = BLOCK_SIZE, block_scales: bool = False) -> int:
        """K and V, every layer: 2 x layers x block_size x KV heads x head_dim x bytes per element (4-bit pools: half a
        byte, and a scale byte for 32 dims), with `block_scales` a byte more per KV head."""
        if dtype == FP4:
            row = config.head_dim // 2 + config.head_dim // FP4_BLOCK
            return 2 * config.num_hidden_layers * block_size * config.num_key_value_heads * row
        elem = torch.tensor([], dtype=dtype).element_size()
        row = block_size * config.head_dim * elem + bool(block_scales)
        return 2 * config.num_hidden_layers * config.num_key_value_heads * row

    @classmethod
    def blocks_for_bytes(cls, config, dtype: torch.dtype, num_bytes: int, block_size: int = BLOCK_SIZE,
                         block_scales: bool = False) -> int:
        return num_bytes // cls.bytes_per_block(config, dtype, block_size, block_scales)

    def step(self, meta) -> PagedStep:
        return PagedStep(self, meta)


def _block_ids(ids):
    """A sequence of block ids as one row of int64 (an array of either kind: a list becomes one in half of numpy's time)."""
    if type(ids) in (list, tuple, range):
        try:
            return array("q", ids)
        except (TypeError, OverflowError):
            raise ValueError("block ids must be one row of whole numbers") from None
    if isinstance(ids, torch.Tensor) and ids.is_cuda:
        raise ValueError("block ids are taken from the host")
    ids = np.asarray(ids)
    if ids.ndim != 1 or ids.size and ids.dtype.kind not in "iu":
        raise ValueError("block ids must be one row of whole numbers")
    return ids.astype(np.int64, copy=False)


def _page_scales(num_blocks: int, hkv: int, device) -> torch.Tensor:
    """e8m0 scales [num_blocks, Hkv] of zeros, in memory that is readable up to the next multiple of four bytes."""
    n = num_blocks * hkv
    whole = torch.zeros(-(-n // 4) * 4, device=device, dtype=torch.uint8)
    return whole[:n].view(torch.float8_e8m0fnu).view(num_blocks, hkv)


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
