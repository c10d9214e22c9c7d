"""Copies of pages within a cache on the GPU (`mllm_copy_pages`, `PagedKVCache.copy_blocks`): bit for bit the pages copied one
by one, in every kind of pool, and nothing else touched."""

import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP8, FP4 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2


def make_cache(kind, hkv, blocks, layers, bs=16, dh=128, seed=0):
    from minillm.cache.paged import PagedKVCache
    from minillm.model.config import LlamaConfig

    cfg = LlamaConfig(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=layers, num_attention_heads=hkv,
                      num_key_value_heads=hkv, head_dim=dh, rms_norm_eps=1e-5, rope_theta=1e4)
    dtype = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp4": FP4}.get(kind, FP8)
    cache = PagedKVCache(cfg, blocks, DEV, dtype, block_size=bs, block_scales=kind == "fp8_blocks")
    g = torch.Generator(device=DEV).manual_seed(seed)
    for t in tensors(cache):
        raw = t.view(torch.uint8)
        raw.copy_(torch.randint(0, 256, raw.shape, generator=g, device=DEV, dtype=torch.uint8))
    return cache


def tensors(cache):
    scaled = cache.fp4 or cache.block_scales
    return [*cache.k, *cache.v, *(cache.k_scale if scaled else ()), *(cache.v_scale if scaled else ())]


def expected(cache, src, dst):
    want = [t.view(torch.uint8).clone() for t in tensors(cache)]
    for w in want:
        w[torch.tensor(dst, device=DEV)] = w[torch.tensor(src, device=DEV)]
    return want


@pytest.mark.parametrize("kind,hkv,blocks,layers,bs,dh,n", [
    ("bf16", 8, 40, 3, 16, 128, 1), ("bf16", 8, 700, 2, 16, 128, 300), ("fp8", 3, 90, 2, 16, 128, 40), ("fp8_blocks", 8, 50, 3, 16, 128, 20),
    ("fp8_blocks", 1, 1200, 1, 16, 128, 513), ("fp8_blocks", 3, 70, 2, 64, 128, 33), ("fp4", 2, 60, 2, 16, 128, 25),
    ("fp4", 5, 60, 1, 32, 192, 20), ("bf16", 1, 33, 70, 16, 64, 16), ("fp32", 1, 30, 1, 16, 20, 10), ("bf16", 1, 20, 1, 1, 2, 7),
    ("fp8", 1, 20, 1, 1, 3, 7)])
def test_copies(hip, kind, hkv, blocks, layers, bs, dh, n):
    cache = make_cache(kind, hkv, blocks, layers, bs, dh)
    rng = random.Random(n)
    ids = list(range(blocks))
    rng.shuffle(ids)
    dst = ids[:n]
    src = [rng.choice(ids[n:]) for _ in range(n)]  # one source may serve several pages
    want = expected(cache, src, dst)
    cache.copy_blocks(src, dst)
    assert all(torch.equal(t.view(torch.uint8), w) for t, w in zip(tensors(cache), want))


def test_copies_go_where_the_pools_are(hip):
    # storage swapped under the same tensor objects between two calls
    cache = make_cache("fp8_blocks", 3, 30, 2)
    cache.copy_blocks([1, 2], [3, 4])
    old = [cache.k[1].data, cache.v_scale[0].data]
    for t in (cache.k[1], cache.v_scale[0]):
        t.data = t.view(torch.uint8).clone().view(t.dtype)
    was = [t.view(torch.uint8).clone() for t in old]
    want = expected(cache, [5, 6], [7, 8])
    cache.copy_blocks([5, 6], [7, 8])
    assert all(torch.equal(t.view(torch.uint8), w) for t, w in zip(tensors(cache), want))
    assert all(torch.equal(t.view(torch.uint8), w) for t, w in zip(old, was))


def test_refused_copies_change_nothing(hip):
    cache = make_cache("fp8_blocks", 2, 9, 2)
    was = [t.view(torch.uint8).clone() for t in tensors(cache)]
    for src, dst in (([1], [9]), ([-1], [2]), ([1, 2], [3, 3]), ([1, 2], [2, 3]), ([4], [4]), ([1, 2], [3])):
        with pytest.raises(ValueError):
            cache.copy_blocks(src, dst)
    with pytest.raises(ValueError, match="host"):
        cache.copy_blocks(torch.tensor([1], device=DEV), [2])
    cache.copy_blocks([], [])
    torch.cuda.synchronize()
    assert all(torch.equal(t.view(torch.uint8), w) for t, w in zip(tensors(cache), was))


def test_replaced_entries_are_seen(hip):
    cache = make_cache("bf16", 2, 9, 2)
    cache.copy_blocks([1], [2])
    cache.k[1] = cache.k[1].clone()
    want = expected(cache, [3], [4])
    cache.copy_blocks([3], [4])
    assert all(torch.equal(t.view(torch.uint8), w) for t, w in zip(tensors(cache), want))


def test_other_stream_and_captured(hip):
    cache = make_cache("fp8_blocks", 8, 60, 2)
    src, dst = list(range(20)), list(range(30, 50))
    side = torch.cuda.Stream()
    want = expected(cache, src, dst)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.copy_blocks(src, dst)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(t.view(torch.uint8), w) for t, w in zip(tensors(cache), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.copy_blocks(dst, list(range(50, 60)) + src[:10])
    for seed in range(3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        for t in tensors(cache):
            t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=g, device=DEV, dtype=torch.uint8))
        want = expected(cache, dst, list(range(50, 60)) + src[:10])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t.view(torch.uint8), w) for t, w in zip(tensors(cache), want))
