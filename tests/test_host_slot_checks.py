"""Every call that appends to a pool with block scales checks the slots it will read, not `append` alone."""

import pytest
import torch

from test_host_long_lived import FP4, FP8, Meta, config

from minillm.attention import hip_backend as hb
from minillm.cache.paged import PagedKVCache


@pytest.mark.parametrize("dtype", [FP8, FP4], ids=["fp8_blocks", "fp4"])
@pytest.mark.parametrize("slots", [torch.zeros(5, dtype=torch.int32), torch.zeros(4, dtype=torch.int64), torch.zeros(10, dtype=torch.int64)[::2],
                                   torch.zeros(5, dtype=torch.int64, device="meta")], ids=["int32", "too_few", "strided", "elsewhere"])
def test_slots(dtype, slots):
    be, bad = hb.HipBackend(), type("Bad", (Meta,), {"slot_mapping": slots})
    cache = PagedKVCache(config(), 3, "cpu", dtype, block_scales=dtype == FP8)
    pools, scales = (cache.k[0], cache.v[0]), cache.scales(0)
    q, k = torch.zeros(5, 4, 128, dtype=torch.bfloat16), torch.zeros(5, 2, 128, dtype=torch.bfloat16)
    cos, w = torch.zeros(5, 128, dtype=torch.bfloat16), torch.ones(128, dtype=torch.bfloat16)
    for call in (lambda: be.forward(q, k, k, *pools, bad, **scales),
                 lambda: be.forward_rotary(q, k, k, cos, cos, *pools, bad, **scales),
                 lambda: be.rope_append(q, k, k, cos, cos, *pools, bad, **scales),
                 lambda: be.rope_append(q, k, k, cos, cos, *pools, bad, qk_norm=(w, w, 1e-5), **scales)):
        with pytest.raises(ValueError, match="slot_mapping"):
            call()
    with pytest.raises(ValueError, match="describe k's tokens"):
        be.append(k, k, *pools, bad, **scales)
