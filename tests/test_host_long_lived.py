"""What long-lived sequences need, without a GPU: 8-bit pools with block scales, copies of pages, forks and compactions, the
rotary forms.  Sizes, host rules and refusals."""

import ctypes
import math
import random
import struct
from pathlib import Path

import pytest
import torch

from minillm import _native
from minillm.attention import hip_backend as hb
from minillm.cache.paged import PagedKVCache
from minillm.cache.prefix import PrefixCache
from minillm.engine.block_manager import BlockManager
from minillm.model import kernels
from minillm.model.config import LLAMA_3_1_8B, LlamaConfig
from minillm.model.rope import attention_factor, compute_inv_freq, rotate

FP8, E8M0, FP4 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.float4_e2m1fn_x2


@pytest.fixture(scope="module", autouse=True)
def library():
    if not _native.LIB_PATH.exists():
        import build_hip

        build_hip.build()


def config(**kw):
    return LlamaConfig(**{**dict(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=2,
                                 num_attention_heads=4, num_key_value_heads=2, head_dim=128, rms_norm_eps=1e-5,
                                 rope_theta=1e4), **kw})


# ------------------------------------------------------------------ 8-bit pools with block scales


def test_block_scaled_cache_shapes_and_bytes():
    cache = PagedKVCache(config(num_key_value_heads=3, num_attention_heads=3), 5, "cpu", FP8, block_size=32, block_scales=True)
    assert cache.block_scales and cache.quantized and not cache.fp4
    assert [tuple(t.shape) for t in (cache.k[1], cache.v[1], cache.k_scale[1], cache.v_scale[1])] == \
        [(5, 32, 3, 128), (5, 32, 3, 128), (5, 3), (5, 3)]
    assert cache.k[0].dtype == FP8 and cache.k_scale[0].dtype == E8M0
    assert cache.scales(1) == {"k_scale": cache.k_scale[1], "v_scale": cache.v_scale[1]}
    # read in dwords: the memory goes on to the next multiple of four
    assert cache.k_scale[0].untyped_storage().nbytes() == 16 and cache.k_scale[0].data_ptr() % 4 == 0
    held = sum(t.view(torch.uint8).numel() for ts in (cache.k, cache.v, cache.k_scale, cache.v_scale) for t in ts)
    assert held == 5 * PagedKVCache.bytes_per_block(config(num_key_value_heads=3), FP8, 32, block_scales=True)
    cfg = LlamaConfig.from_dict(LLAMA_3_1_8B)
    assert PagedKVCache.bytes_per_block(cfg, FP8, block_scales=True) == PagedKVCache.bytes_per_block(cfg, FP8) + 2 * 32 * 8
    assert PagedKVCache.blocks_for_bytes(cfg, FP8, 2 ** 30, block_scales=True) == 2 ** 30 // (2 ** 20 + 512)


def test_block_scaled_cache_refusals():
    for kw, match in ((dict(dtype=torch.bfloat16), "float8_e4m3fn"), (dict(dtype=FP4), "float8_e4m3fn"),
                      (dict(cfg=config(head_dim=64)), "head_dim of 128"), (dict(block_size=8), "16, 32 or 64"),
                      (dict(block_size=128), "16, 32 or 64"), (dict(block_size=48), "16, 32 or 64"),
                      (dict(k_scale=0.5), "not with block_scales"), (dict(v_scale=2.0), "not with block_scales")):
        kw = {**dict(cfg=config(), dtype=FP8, block_size=16), **kw}
        with pytest.raises(ValueError, match=match):
            PagedKVCache(kw.pop("cfg"), 3, "cpu", kw.pop("dtype"), block_scales=True, **kw)
    cache = PagedKVCache(config(), 3, "cpu", FP8, block_scales=True)
    slots = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        cache.read(0, slots)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        cache.read(0, slots, torch.float32)


def test_pool_type_goes_by_the_scales():
    cache = PagedKVCache(config(), 3, "cpu", FP8, block_scales=True)
    assert hb.pool_type(cache.k[0]) == hb.pool_type(cache.k[0], 0.5) == _native.POOL_FP8
    assert hb.pool_type(cache.k[0], torch.tensor(0.5)) == _native.POOL_FP8  # a tensor of one per-tensor scale
    assert hb.pool_type(cache.k[0], cache.k_scale[0]) == _native.POOL_FP8_BLOCKS
    ks, vs = cache.k_scale[0], cache.v_scale[0]
    hb.check_scales(cache.k[0], ks, vs)
    for bad in ((ks, 1.0), (ks, vs.view(torch.uint8)), (ks[:2], vs), (ks, vs.t().contiguous()), (ks, vs.t()), (ks, vs.to("meta"))):
        with pytest.raises(ValueError, match="scale"):
            hb.check_scales(cache.k[0], *bad)


class Meta:
    block_size, query_start_loc = 16, [0, 5]
    slot_mapping = torch.zeros(5, dtype=torch.int64)


def test_backend_refusals():
    be = hb.HipBackend()
    cache = PagedKVCache(config(), 3, "cpu", FP8, block_scales=True)
    kc, vc, scales = cache.k[0], cache.v[0], cache.scales(0)
    q, k = torch.zeros(5, 4, 128, dtype=torch.bfloat16), torch.zeros(5, 2, 128, dtype=torch.bfloat16)
    cos = torch.zeros(5, 128, dtype=torch.bfloat16)
    for args in ((q.float(), k.float(), k.float()), (q, k.half(), k)):
        with pytest.raises(ValueError, match="fp8 pool, q, k and v"):
            be.forward(*args, kc, vc, Meta, **scales)
    with pytest.raises(ValueError, match="v_scale"):
        be.forward(q, k, k, kc, vc, Meta, k_scale=scales["k_scale"])
    with pytest.raises(ValueError, match="one device"):
        be.forward(q.to("meta"), k, k, kc, vc, Meta, **scales)
    with pytest.raises(ValueError, match="one device"):
        be.forward_rotary(q, k, k, cos.to("meta"), cos.to("meta"), kc, vc, Meta, **scales)
    with pytest.raises(ValueError, match="of one dtype"):
        be.append(k[..., :64], k[..., :64], kc, vc, Meta, **scales)
    with pytest.raises(ValueError, match="describe k's tokens"):
        be.append(k[:3], k[:3], kc, vc, Meta, **scales)
    for slots in (Meta.slot_mapping.int(), torch.zeros(10, dtype=torch.int64)[::2], Meta.slot_mapping.to("meta")):
        bad = type("Bad", (Meta,), {"slot_mapping": slots})
        with pytest.raises(ValueError, match="describe k's tokens"):
            be.append(k, k, kc, vc, bad, **scales)
    with pytest.raises(ValueError, match="K and V alike"):
        be.forward(q, k, k, kc, vc, Meta, v_scale=scales["v_scale"])
    with pytest.raises(ValueError, match="alike"):
        be.append(k, k, kc, vc[:2], Meta, **scales)
    for kw, match in ((dict(q=q[:3]), "N, H, Dh"), (dict(q=q[:, :3]), "N, H, Dh"), (dict(q=q[..., :64]), "N, H, Dh"),
                      (dict(out=q.float()), "out must be like q"), (dict(vc=vc[:2]), "alike"),
                      (dict(vc=torch.zeros_like(vc, dtype=torch.bfloat16)), "alike"), (dict(out=q.to("meta")), "one device")):
        a = dict(q=q, vc=vc, out=torch.empty_like(q)) | kw
        with pytest.raises(ValueError, match=match):
            be.attend(a["q"], kc, a["vc"], Meta, a["out"], **scales)
    p16 = torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="fp8 pools only"):
        be.forward(q, k, k, p16, p16.clone(), Meta, **scales)


def test_entry_points_check_their_arguments():
    lib, a = _native.lib(), 1 << 20

    def append(k=a, st=256, n=1, nb=4, bs=16, hkv=2, dh=128, dtype=2, scales=a, slots=a):
        lib.call("mllm_kv_append_fp8_blocks", k, st, 128, a, 256, 128, dtype, a, a, scales, a, nb, bs, hkv, dh, slots, n, None)

    for kw, match in ((dict(dtype=0), "dtype"), (dict(n=-1), "sizes"), (dict(hkv=0), "sizes"), (dict(dh=64), "head_dim"),
                      (dict(bs=8), "block_size"), (dict(bs=48), "block_size"), (dict(bs=128), "block_size"),
                      (dict(nb=1 << 31), "too large"), (dict(n=1 << 40), "too many"), (dict(k=None), "null"),
                      (dict(scales=None), "null"), (dict(slots=None), "null"), (dict(k=a + 2), "aligned"), (dict(st=257), "aligned")):
        with pytest.raises(ValueError, match=match):
            append(**kw)
    append(n=0, k=None)

    def read(n=1, dtype=2, out=a, bs=16, slots=a):
        lib.call("mllm_kv_read_fp8_blocks", a, a, a, a, 4, bs, 2, 128, slots, n, dtype, out, a, None)

    for kw, match in ((dict(dtype=0), "dtype"), (dict(bs=24), "block_size"), (dict(out=a + 2), "aligned"), (dict(slots=None), "null")):
        with pytest.raises(ValueError, match=match):
            read(**kw)
    read(n=0, slots=None)

    def decode(work=4, merges=0, scales=a, dh=128, h=8, bs=16, split=8, q=a):
        lib.call("mllm_paged_decode_fp8_blocks", q, 1024, 128, a, a, scales, a, 4, bs, h, 2, dh, a, a, a, work, a, merges, split,
                 0.1, 2, a, 1024, 128, None, 0, None)

    for kw, match in ((dict(dh=64), "head_dim"), (dict(h=7), "multiple"), (dict(h=64), "at most 16"), (dict(bs=24), "block_size"),
                      (dict(split=0), "pages_per_split"), (dict(merges=1), "workspace"), (dict(scales=a + 2), "aligned"),
                      (dict(scales=None), "null"), (dict(q=a + 8), "aligned")):
        with pytest.raises(ValueError, match=match):
            decode(**kw)
    decode(work=0)
    for scales, match in ((None, "null"), (a + 1, "aligned")):
        with pytest.raises(ValueError, match=match):
            lib.call("mllm_paged_prefill_fp8_blocks", a, 1024, 128, a, a, scales, a, 4, 16, 8, 2, 128, a, a, a, a, a, 1, 32, 0.1,
                     2, a, 1024, 128, None)


# ------------------------------------------------------------------ copies of pages


@pytest.mark.parametrize("kind", ["bf16", "fp8", "fp8_blocks", "fp4"])
def test_copy_blocks_on_the_host(kind):
    dtype = {"bf16": torch.bfloat16, "fp4": FP4}.get(kind, FP8)
    cache = PagedKVCache(config(), 9, "cpu", dtype, block_scales=kind == "fp8_blocks")
    lists = [cache.k, cache.v] + ([cache.k_scale, cache.v_scale] if kind in ("fp8_blocks", "fp4") else [])
    for ts in lists:
        for t in ts:
            t.view(torch.uint8).copy_(torch.randint(0, 256, t.view(torch.uint8).shape, dtype=torch.uint8))
    before = [[t.view(torch.uint8).clone() for t in ts] for ts in lists]
    cache.copy_blocks([3, 3, 8], (0, 5, 1))
    for ts, was in zip(lists, before):
        for t, w in zip(ts, was):
            w[torch.tensor([0, 5, 1])] = w[torch.tensor([3, 3, 8])]
            assert torch.equal(t.view(torch.uint8), w)
    cache.copy_blocks([], [])
    cache.copy_blocks(torch.tensor([2]), range(4, 5))


def test_copy_blocks_refusals():
    cache = PagedKVCache(config(), 9, "cpu", torch.bfloat16)
    for src, dst, match in (([1], [9], "outside"), ([-1], [2], "outside"), ([1, 2], [3, 3], "written twice"),
                            ([1, 2], [2, 3], "read and written"), ([4], [4], "read and written"), ([1, 2], [3], "2 blocks"),
                            ([1.0], [2], "whole numbers"), ([[1]], [[2]], "one row"), ([1 << 63], [2], "whole numbers"),
                            (torch.tensor([1.0]), [2], "whole numbers"), (torch.tensor([[1]]), [2], "one row")):
        with pytest.raises(ValueError, match=match):
            cache.copy_blocks(src, dst)
    cache.k[0] = torch.zeros(8, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="9 blocks"):
        cache.copy_blocks([1], [2])


def test_copy_pages_checks_its_arguments():
    lib, q = _native.lib(), struct.pack

    def call(tensors=q("2Q", 1 << 20, 1 << 21), nbytes=q("2q", 4096, 8), n=2, pages=9, src=q("2q", 1, 2), dst=q("2q", 3, 4), pairs=2):
        lib.call("mllm_copy_pages", tensors, nbytes, n, pages, src, dst, pairs, None)

    for kw, match in ((dict(n=-1), "sizes"), (dict(pairs=-1), "sizes"), (dict(pages=1 << 31), "too many"), (dict(src=None), "null"),
                      (dict(tensors=None), "null"), (dict(tensors=q("2Q", 1 << 20, 0)), "null"), (dict(nbytes=q("2q", 4096, 0)), "page"),
                      (dict(nbytes=q("2q", 1 << 23, 8)), "page too large"), (dict(src=q("2q", 1, 9)), "block 9 is outside"),
                      (dict(dst=q("2q", -1, 2)), "block -1 is outside"), (dict(dst=q("2q", 5, 5)), "written twice"),
                      (dict(dst=q("2q", 2, 5)), "read and written"), (dict(pages=0), "outside")):
        with pytest.raises(ValueError, match=match):
            call(**kw)
    call(pairs=0, src=None)
    call(n=0, tensors=None)


def test_copies_follow_pools_that_moved():
    cache = PagedKVCache(config(head_dim=128), 6, "cpu", FP8, block_scales=True)
    before = cache._page_tensors()
    assert cache._page_tensors() is not None and cache._page_tensors() == before
    kept = cache.v[1].data
    cache.v[1].data = kept.clone()  # the same tensor object over other memory
    cache.k_scale[0] = cache.k_scale[0].view(torch.uint8).clone().view(torch.float8_e8m0fnu)
    after = cache._page_tensors()
    pointers = struct.unpack(f"{after[2]}Q", after[0])
    assert pointers == tuple(t.data_ptr() for t in (*cache.k, *cache.v, *cache.k_scale, *cache.v_scale))
    assert pointers != struct.unpack(f"{before[2]}Q", before[0])
    cache.k[0] = cache.k[0][1:]
    with pytest.raises(ValueError, match="of 6 blocks"):
        cache.check_pages()


def test_nothing_is_taken_where_pages_cannot_be_copied():
    from minillm.engine.core import AddRequest

    core = engine()
    core.add_request(AddRequest("a", list(range(3, 23)), 8))
    core.step()
    core.cache.v[0] = core.cache.v[0].transpose(0, 1)
    free, running = core.blocks.num_free, list(core.scheduler.running)
    for call in (lambda: core.fork("a", "b"), core.compact):
        with pytest.raises(ValueError, match="contiguous"):
            call()
    assert core.blocks.num_free == free and core.scheduler.running == running


# ------------------------------------------------------------------ forks, trims, compactions


def test_fork_shares_full_blocks_and_copies_the_last():
    blocks = BlockManager(10, 16)
    table = blocks.allocate(4)  # 0 .. 3
    child, copies = blocks.fork(table, 40)  # two full blocks and 8 tokens of the third
    assert child[:2] == table[:2] and len(child) == 3 and copies == [(table[2], child[2])] and child[2] not in table
    blocks.check([table, child])
    even, none = blocks.fork(table, 32)
    assert even == table[:2] and none == []
    roomy, copies = blocks.fork(table, 40, reserve_tokens=70)
    assert len(roomy) == 5 and copies == [(table[2], roomy[2])]
    blocks.check([table, child, even, roomy])
    with pytest.raises(ValueError, match="does not hold"):
        blocks.fork(table, 65)
    held = [list(table), list(child), list(even), list(roomy)]
    with pytest.raises(RuntimeError, match="free"):
        blocks.fork(table, 40, reserve_tokens=16 * 9)
    blocks.check(held)  # nothing was taken
    blocks.trim(roomy, 33)
    assert len(roomy) == 3
    blocks.trim(roomy, 100)
    assert len(roomy) == 3
    blocks.check([table, child, even, roomy])
    for t in (table, child, even, roomy):
        blocks.free(t)
    blocks.check([])
    assert blocks.num_free == 10


def test_trim_to_nothing():
    blocks = BlockManager(4, 16)
    table = blocks.allocate(3)
    blocks.trim(table, 0)
    assert table == [] and blocks.num_free == 4
    empty, copies = blocks.fork(table, 0)
    assert empty == [] and copies == []
    blocks.check([table, empty])


@pytest.mark.parametrize("seed", range(6))
def test_compact_moves_everything_to_the_front(seed):
    # a model of the pool: what each block holds and which name it carries follow the moves, the order of eviction stays
    rng = random.Random(seed)
    prefix = PrefixCache()
    blocks = BlockManager(60, 16, prefix)
    tables, holds = [], {}
    for i in range(40):
        if rng.random() < 0.6 and blocks.num_free >= 6:
            t = blocks.allocate(rng.randint(1, 6))
            for b in t:
                holds[b] = (i, b)
                if rng.random() < 0.5:
                    prefix.insert(b"%d-%d" % (i, b), b)
            tables.append(t)
        elif tables:
            blocks.free(tables.pop(rng.randrange(len(tables))))
        if tables and rng.random() < 0.2:
            shared = list(rng.choice(tables))
            blocks.acquire(shared)
            tables.append(shared)
    order = [(name, b) for t, (tier, b) in sorted(blocks._live()) if tier == 1 for name in [prefix._name_by_block[b]]]
    names = {n: holds[b] for n, b in prefix._block_by_name.items()}
    free, cached = blocks.num_free, blocks.num_cached
    moves = blocks.compact()
    assert not {a for a, _ in moves} & {b for _, b in moves} and len({b for _, b in moves}) == len(moves)
    to = dict(moves)
    for a, b in moves:
        holds[b] = holds[a]
    tables = [[to.get(b, b) for b in t] for t in tables]
    used = blocks.num_blocks - blocks.num_free + blocks.num_cached
    assert all(b < used for t in tables for b in t) and all(b < used for b in prefix._block_by_name.values())
    assert {n: holds[b] for n, b in prefix._block_by_name.items()} == names
    assert [prefix._name_by_block[b] for n, b in prefix._block_by_name.items()] == list(prefix._block_by_name)
    blocks.check(tables)
    assert (blocks.num_free, blocks.num_cached) == (free, cached)
    assert [(prefix._name_by_block[b]) for t, (tier, b) in sorted(blocks._live()) if tier == 1] == [n for n, _ in order]
    assert blocks.compact() == []
    taken = blocks.allocate(blocks.num_free - blocks.num_cached)  # blank ones first: none is in use
    assert not set(taken) & {b for t in tables for b in t} and not set(taken) & set(prefix._block_by_name.values())
    blocks.allocate(blocks.num_free)
    assert blocks.num_free == 0 and blocks.num_cached == 0


# ------------------------------------------------------------------ rotary forms


def test_reference_rope_stays():
    cfg = LlamaConfig.from_dict(LLAMA_3_1_8B)
    assert cfg.rope_by_table and cfg.rotary_dim == 128 and attention_factor(cfg) == 1.0
    assert config(rope_scaling={"rope_type": "linear", "factor": 2.0}).rope_by_table
    for kw in (dict(rope_interleaved=True), dict(partial_rotary_factor=0.5)):
        assert not config(**kw).rope_by_table
    with pytest.raises(ValueError, match="even number"):
        config(head_dim=64, partial_rotary_factor=0.36).rotary_dim
    with pytest.raises(ValueError, match="even number"):
        config(partial_rotary_factor=0.0).rotary_dim
    with pytest.raises(NotImplementedError, match="dynamic"):
        compute_inv_freq(config(rope_scaling={"rope_type": "dynamic", "factor": 2.0}))


def test_config_keys_of_the_forms():
    base = dict(vocab_size=256, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, rms_norm_eps=1e-5)
    cfg = LlamaConfig.from_dict(base)
    assert not cfg.rope_interleaved and cfg.partial_rotary_factor == 1.0
    cfg = LlamaConfig.from_dict({**base, "rope_interleaved": True, "partial_rotary_factor": 0.5})
    assert cfg.rope_interleaved and cfg.rotary_dim == 8
    cfg = LlamaConfig.from_dict({**base, "rope_interleave": True, "rope_parameters": {"rope_theta": 1e4, "partial_rotary_factor": 0.25}})
    assert cfg.rope_interleaved and cfg.rotary_dim == 4
    for none in ({"partial_rotary_factor": None}, {"rope_parameters": {"rope_theta": 1e4, "partial_rotary_factor": None}}):
        assert LlamaConfig.from_dict({**base, **none}).partial_rotary_factor == 1.0


@pytest.mark.parametrize("rope", [
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096},
    {"rope_type": "yarn", "factor": 2.5, "original_max_position_embeddings": 8192, "beta_fast": 20.0, "beta_slow": 2.0},
    {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096, "mscale": 0.7, "mscale_all_dim": 1.3},
    {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 2048, "attention_factor": 1.25},
], ids=["linear", "yarn", "yarn-betas", "yarn-mscale", "yarn-factor"])
def test_scaled_frequencies_match_transformers(rope):
    transformers = pytest.importorskip("transformers")
    from transformers.models.llama.modeling_llama import LlamaRotaryEmbedding

    hf = transformers.LlamaConfig(vocab_size=256, hidden_size=512, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
                                  num_key_value_heads=2, max_position_embeddings=65536, rope_parameters={**rope, "rope_theta": 10000.0})
    cfg = LlamaConfig.from_dict(hf.to_dict())
    theirs = LlamaRotaryEmbedding(hf)
    torch.testing.assert_close(compute_inv_freq(cfg), theirs.inv_freq.float(), rtol=1e-5, atol=0)
    assert attention_factor(cfg) == pytest.approx(theirs.attention_scaling, rel=1e-6)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("rot", [32, 16, 6, 2])
def test_rotate_against_complex_numbers(interleaved, rot):
    g = torch.Generator().manual_seed(rot)
    x = torch.randn(2, 3, 5, 32, generator=g, dtype=torch.float64)
    pos = torch.randint(0, 100000, (2, 5), generator=g)
    inv = torch.rand(rot // 2, generator=g)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    turn = torch.polar(torch.full((2, 1, 5, rot // 2), 1.25, dtype=torch.float64), pos[:, None, :, None].double() * inv.double())
    z = torch.complex(x[..., a], x[..., b]) * turn
    want = x.clone()
    want[..., a], want[..., b] = z.real, z.imag
    torch.testing.assert_close(rotate(x, pos, inv, interleaved, 1.25), want, rtol=1e-12, atol=1e-12)


def test_rotate_has_gradients():
    x = torch.randn(1, 2, 3, 8, dtype=torch.float64, requires_grad=True)
    pos, inv = torch.tensor([[0, 5, 7]]), torch.tensor([0.5, 0.1])
    assert torch.autograd.gradcheck(lambda y: rotate(y, pos, inv, True, 1.5), (x,))


def test_rotary_refusals():
    q, k = torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
    pos, inv = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(32)
    for kw, match in ((dict(k=k[:1]), "k must be"), (dict(k=k[..., :32]), "k must be"), (dict(k=k[:, :0]), "k must be"),
                      (dict(positions=pos[:1]), "positions"), (dict(positions=pos.int()), "positions"),
                      (dict(inv_freq=inv.double()), "inv_freq"), (dict(inv_freq=torch.zeros(33)), "inv_freq"),
                      (dict(inv_freq=torch.zeros(0)), "inv_freq"), (dict(k=k.half()), "one dtype"),
                      (dict(positions=pos.to("meta")), "one device"), (dict(), "on a GPU")):
        a = dict(q=q, k=k, positions=pos, inv_freq=inv) | kw
        with pytest.raises(ValueError, match=match):
            kernels.rotary(**a)

    lib, a = _native.lib(), 1 << 20

    def call(q=a, pairs=64, b=1, t=1, h=4, dh=128, dtype=2, pos=a):
        args = _native.RotaryArgs(q=q, k=a, q_sb=512, q_sh=128, q_st=512, k_sb=256, k_sh=128, k_st=256, positions=pos, p_sb=1, p_st=1,
                                  inv_freq=a, q_out=a, k_out=a, qo_sb=512, qo_sh=128, qo_st=512, ko_sb=256, ko_sh=128, ko_st=256,
                                  factor=1.0, pairs=pairs, interleaved=0, batch=b, seq=t, num_heads=h, num_kv_heads=2, head_dim=dh,
                                  dtype=dtype)
        lib.call("mllm_rotary", ctypes.addressof(args), None)

    for kw, match in ((dict(dtype=0), "dtype"), (dict(t=-1), "sizes"), (dict(h=0), "sizes"), (dict(pairs=65), "pairs"),
                      (dict(pairs=0), "pairs"), (dict(pairs=513, dh=2048), "too long"), (dict(dh=8192), "too long"),
                      (dict(q=None), "null"), (dict(pos=None), "null"), (dict(q=a + 1), "misaligned"),
                      (dict(b=1 << 16, t=1 << 16), "sizes")):
        with pytest.raises(ValueError, match=match):
            call(**kw)
    call(t=0, q=None)
    with pytest.raises(ValueError, match="null arguments"):
        lib.call("mllm_rotary", None, None)


def test_rotary_args_match_the_header(tmp_path):
    import subprocess

    fields = [name for name, _ in _native.RotaryArgs._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "minillm_hip.h"\nint main(void) {\n'
                   + 'printf("%zu\\n", sizeof(mllm_rotary_args));\n'
                   + "".join(f'printf("%zu\\n", offsetof(mllm_rotary_args, {f}));\n' for f in fields) + "return 0;\n}\n")
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", "-std=c99", f"-I{include}", str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_native.RotaryArgs)] + [getattr(_native.RotaryArgs, f).offset for f in fields]


@pytest.mark.parametrize("rope", [{"rope_type": "linear", "factor": 4.0},
                                  {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}])
def test_scaled_tables_on_the_host(rope):
    # angles of far positions in float64, whatever the table's type; the plain and the llama3 tables as they were
    from minillm.model.llama import RotaryEmbedding

    cfg = config(rope_scaling=rope)
    pos = torch.tensor([[0, 5, 999983, 123456789]])
    for dtype in (torch.float64, torch.float32, torch.bfloat16):
        cos, sin = RotaryEmbedding(cfg)(pos, dtype)
        ang = pos[..., None].double() * compute_inv_freq(cfg).double()
        for got, f in ((cos, torch.cos), (sin, torch.sin)):
            assert got.dtype == dtype and torch.equal(got, (f(torch.cat([ang, ang], -1)) * attention_factor(cfg)).to(dtype))
    plain = RotaryEmbedding(config())
    cos, _ = plain(pos, torch.float32)
    ang = pos[..., None].float() * compute_inv_freq(config())
    assert torch.equal(cos, torch.cat([ang, ang], -1).cos())


@pytest.mark.parametrize("kw", [dict(rope_interleaved=True), dict(partial_rotary_factor=0.5),
                                dict(rope_interleaved=True, partial_rotary_factor=0.5, rope_scaling={
                                    "rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64})])
def test_model_on_the_host_rotates_by_position(kw):
    # a contiguous forward pass on the CPU through a backend in torch operations: equal to the attention by hand
    from minillm.attention.base import AttentionBackend
    from minillm.model.llama import LlamaAttention

    seen = {}

    class Plain(AttentionBackend):
        def prefill(self, q, k, v, key_valid=None, **_):
            seen.update(q=q, k=k)
            return torch.zeros_like(q)

        def forward(self, *args):
            raise AssertionError

    cfg = config(hidden_size=32, head_dim=16, **kw)
    attn = LlamaAttention(cfg, Plain(), 0)
    x, pos, inv = torch.randn(2, 5, 32), torch.arange(5).expand(2, 5), compute_inv_freq(cfg)
    attn(x, pos, inv)
    for name, proj in (("q", attn.q_proj), ("k", attn.k_proj)):
        y = proj(x).view(2, 5, -1, 16).transpose(1, 2)
        torch.testing.assert_close(seen[name], rotate(y, pos, inv, cfg.rope_interleaved, attention_factor(cfg)))
    seen["q"].sum().backward()
    assert attn.q_proj.weight.grad is not None and math.isfinite(attn.q_proj.weight.grad.sum().item())


# ------------------------------------------------------------------ the engine: forks and compactions


def engine(num_kv_blocks=40, max_batch_size=6, **kw):
    """A small float32 model on the CPU behind the oracle's attention, picking the best token, or, for requests whose name
    ends in "+", the second best."""
    from minillm.engine.core import EngineCore
    from minillm.model.llama import LlamaForCausalLM, random_init_
    from oracle_engine import OracleBackend, oracle_metadata

    cfg = config(vocab_size=97, hidden_size=32, num_attention_heads=4, num_key_value_heads=2, head_dim=8, max_position_embeddings=256)
    model = random_init_(LlamaForCausalLM(cfg, OracleBackend()), std=0.3, seed=5)

    def sampler(reqs, logits):
        best = logits.topk(2, dim=-1).indices
        return [int(best[i, 1 if r.req_id.endswith("+") else 0]) for i, r in enumerate(reqs)]

    return EngineCore(model, metadata_builder=oracle_metadata, sampler=sampler, max_batch_size=max_batch_size,
                      num_kv_blocks=num_kv_blocks, **kw)


def drain(core, outs, each=None):
    while core.has_work():
        for o in core.step().outputs:
            outs.setdefault(o.req_id, []).extend(o.new_token_ids)
        core.check_blocks()
        if each is not None:
            each(core)
    return outs


@pytest.mark.parametrize("chunked", [False, True])
@pytest.mark.parametrize("at", [3, 12])
def test_a_fork_goes_on_as_its_own_request_would(chunked, at):
    from minillm.engine.core import AddRequest

    prompt, n = list(range(3, 3 + 21)), 24
    core, outs = engine(chunked_prefill=chunked, max_num_batched_tokens=8 if chunked else None), {}
    core.add_request(AddRequest("a", prompt, n))
    core.add_request(AddRequest("other", prompt[:5], 9))
    while len(outs.get("a", [])) < at:
        for o in core.step().outputs:
            outs.setdefault(o.req_id, []).extend(o.new_token_ids)
    used = core.blocks.num_blocks - core.blocks.num_free
    core.fork("a", "b+", max_tokens=n - 2)
    assert core.blocks.num_blocks - core.blocks.num_free <= used + 1  # full blocks are shared
    core.check_blocks()
    drain(core, outs)
    assert len(outs["a"]) == n and len(outs["b+"]) == n - 2 - at
    alone = engine()
    alone.add_request(AddRequest("a", prompt, n))
    alone.add_request(AddRequest("b+", prompt + outs["a"][:at], n - 2 - at))
    want = drain(alone, {})
    assert outs["a"] == want["a"] and outs["b+"] == want["b+"] and outs["b+"] != outs["a"][at:n - 2]
    assert core.blocks.num_free == core.blocks.num_blocks


def test_fork_within_a_prompt_and_refusals():
    from minillm.engine.core import AddRequest

    core, outs = engine(chunked_prefill=True, max_num_batched_tokens=10, max_batch_size=2), {}
    prompt = list(range(3, 3 + 35))
    core.add_request(AddRequest("a", prompt, 6))
    with pytest.raises(ValueError, match="no running request"):
        core.fork("a", "b")
    core.step()  # ten of 35 tokens
    for bad in (("x", "b"), ("a", "a")):
        with pytest.raises(ValueError):
            core.fork(*bad)
    with pytest.raises(ValueError, match="leaves none"):
        core.fork("a", "b", max_tokens=0)
    with pytest.raises(ValueError, match="max_model_len"):
        core.fork("a", "b", max_tokens=1000)
    core.fork("a", "b")
    with pytest.raises(RuntimeError, match="run already"):
        core.fork("a", "c")
    drain(core, outs)
    assert outs["a"] == outs["b"] and len(outs["a"]) == 6


def test_fork_of_a_full_pool_is_refused_and_changes_nothing():
    from minillm.engine.core import AddRequest

    core, outs = engine(num_kv_blocks=2, enable_prefix_caching=False), {}
    core.add_request(AddRequest("a", list(range(3, 23)), 8))
    core.step()
    with pytest.raises(RuntimeError, match="free"):
        core.fork("a", "b")
    core.check_blocks()
    assert len(drain(core, outs)["a"]) == 7


def test_compaction_between_steps_changes_no_token():
    from minillm.engine.core import AddRequest

    runs = []
    for compacts in (False, True):
        core, outs = engine(num_kv_blocks=30), {}
        rng = random.Random(4)
        ps = [[rng.randrange(3, 97) for _ in range(rng.randrange(4, 60))] for _ in range(9)]
        ps[5] = ps[1] + [7, 8]  # a shared head
        for i, p in enumerate(ps):
            core.add_request(AddRequest("r%d" % i, p, 5 + 3 * i))
        moved = []

        def each(core):
            if compacts:
                n = core.compact()
                held = {b for r in core.scheduler.running for b in r.block_ids}
                assert all(b < n for b in held) and n == core.blocks.num_blocks - core.blocks.num_free + core.blocks.num_cached
                core.check_blocks()
                moved.append(n)

        runs.append(drain(core, outs, each))
        assert not compacts or len(set(moved)) > 3
    assert runs[0] == runs[1]
