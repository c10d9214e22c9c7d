"""`PagedKVCache.read` of pools with block scales checks what the kernel goes by: entries a program has replaced."""

import pytest
import torch

from test_host_long_lived import FP4, FP8, config

from minillm.cache.paged import PagedKVCache


@pytest.mark.parametrize("dtype", [FP8, FP4], ids=["fp8_blocks", "fp4"])
def test_replaced_entries(dtype):
    slots = torch.zeros(2, dtype=torch.int64)
    make = lambda: PagedKVCache(config(), 6, "cpu", dtype, block_scales=dtype == FP8)
    cache = make()
    with pytest.raises(RuntimeError, match="GPU"):
        cache.read(0, slots)
    for scales in ("k_scale", "v_scale"):
        for bad in (lambda s: s[:4], lambda s: s.view(torch.uint8), lambda s: 0.5, lambda s: s.transpose(0, 1),
                    lambda s: s.to("meta")):
            cache = make()
            held = getattr(cache, scales)
            held[0] = bad(held[0])
            with pytest.raises(ValueError, match="scale"):
                cache.read(0, slots)
    for bad in (lambda p: p[:4], lambda p: p.transpose(1, 2), lambda p: p.view(torch.uint8)):
        cache = make()
        cache.v[0] = bad(cache.v[0])
        with pytest.raises(ValueError, match="alike and contiguous"):
            cache.read(0, slots)
    cache = make()
    cache.k[0], cache.v[0] = (p.transpose(0, 1) for p in (cache.k[0], cache.v[0]))
    with pytest.raises(ValueError, match="alike and contiguous"):
        cache.read(0, slots)
