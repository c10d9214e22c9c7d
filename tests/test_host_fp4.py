"""4-bit pools and head norms without a GPU: sizes, host rules and refusals."""

import ctypes

import pytest
import torch

from minillm import _native
from minillm.attention import hip_backend as hb
from minillm.cache.paged import PagedKVCache
from minillm.model.config import LLAMA_3_1_8B, LlamaConfig

FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


@pytest.fixture(scope="module", autouse=True)
def library():
    if not _native.LIB_PATH.exists():
        import build_hip

        build_hip.build()


def config(**kw):
    return LlamaConfig(**{**dict(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=2,
                                 num_attention_heads=4, num_key_value_heads=2, head_dim=128, rms_norm_eps=1e-5,
                                 rope_theta=1e4), **kw})


def test_cache_shapes_and_bytes():
    cache = PagedKVCache(config(), 3, "cpu", FP4, block_size=32)
    assert cache.fp4 and not cache.quantized
    assert [tuple(t.shape) for t in (cache.k[1], cache.v[1], cache.k_scale[1], cache.v_scale[1])] == \
        [(3, 32, 2, 64), (3, 32, 2, 64), (3, 32, 4, 2), (3, 2, 4, 32)]
    assert cache.k[0].dtype == FP4 and cache.v_scale[0].dtype == E8M0
    assert cache.scales(1) == {"k_scale": cache.k_scale[1], "v_scale": cache.v_scale[1]}
    assert cache.scales(0)["k_scale"].data_ptr() != cache.scales(1)["k_scale"].data_ptr()
    held = sum(t.view(torch.uint8).numel() for ts in (cache.k, cache.v, cache.k_scale, cache.v_scale) for t in ts)
    assert held == 3 * PagedKVCache.bytes_per_block(config(), FP4, 32)
    cfg = LlamaConfig.from_dict(LLAMA_3_1_8B)
    assert PagedKVCache.bytes_per_block(cfg, FP4) == 32 * 17 * 2 ** 10
    assert PagedKVCache.blocks_for_bytes(cfg, FP4, 2 ** 30) == 2 ** 30 // (32 * 17 * 2 ** 10)


def test_cache_refusals():
    with pytest.raises(ValueError, match="multiple of 64"):
        PagedKVCache(config(head_dim=96), 3, "cpu", FP4)
    with pytest.raises(ValueError, match="fp8 pools only"):
        PagedKVCache(config(), 3, "cpu", FP4, k_scale=0.5)
    cache = PagedKVCache(config(), 3, "cpu", FP4)
    slots = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        cache.read(0, slots)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        cache.read(0, slots, torch.float32)
    for bad in (slots.int(), slots[None]):
        with pytest.raises(ValueError, match="int64"):
            cache.read(0, bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float8_e4m3fn])
def test_read_of_other_pools(dtype):
    cache = PagedKVCache(config(), 4, "cpu", dtype, **({"k_scale": 0.5, "v_scale": 2.0} if dtype.itemsize == 1 else {}))
    k, v = torch.randn(2, 4, 16, 2, 128).unbind(0)
    cache.k[1].copy_(k)
    cache.v[1].copy_(v)
    slots = torch.tensor([63, 0, 17, 17])
    got_k, got_v = cache.read(1, slots)
    fp8 = dtype == torch.float8_e4m3fn
    assert got_k.dtype == got_v.dtype == (torch.bfloat16 if fp8 else dtype)
    for got, x, s in ((got_k, k, 0.5), (got_v, v, 2.0)):
        want = x.to(dtype).float() * (s if fp8 else 1.0)
        assert torch.equal(got, want.flatten(0, 1)[slots].to(got.dtype))
    # a step's padding rows have no slot
    for got in cache.read(1, torch.tensor([-1, 5, 64])):
        assert bool((got[::2] == 0).all()) and bool((got[1] != 0).any())


def test_split_sizes_of_4bit_pools():
    assert hb.fp4_heads(32, 8) == 2 and hb.fp4_heads(16, 2) == 2 and hb.fp4_heads(16, 1) == 1
    assert hb.fp4_heads(40, 8) == 2 and hb.fp4_heads(12, 4) == 2 and hb.fp4_heads(15, 5) == 1 and hb.fp4_heads(96, 8) == 1
    for heads, kv in ((32, 8), (16, 2), (8, 8), (16, 1)):
        for pages in (1, 5, 100, 4096, 34000, 300000):
            c = hb.pages_per_split(pages, kv, heads, kv_fp4=True)
            assert hb.MIN_SPLIT_PAGES <= c <= hb.MAX_SPLIT_PAGES
            records, _ = hb.decode_plan_size(pages, 3, c)
            assert records <= hb.decode_records_bound(pages, 3, kv, heads, kv_fp4=True) or pages > 4096


def test_scales_are_checked():
    cache = PagedKVCache(config(), 3, "cpu", FP4)
    k, ks, vs = cache.k[0], cache.k_scale[0], cache.v_scale[0]
    hb.check_scales(k, ks, vs)
    for bad in ((1.0, 1.0), (ks.view(torch.uint8), vs), (ks[:2], vs), (ks, ks), (vs, vs), (ks, vs.transpose(2, 3))):
        with pytest.raises(ValueError, match="scale"):
            hb.check_scales(k, *bad)


class Meta:
    block_size, query_start_loc = 16, [0, 5]
    slot_mapping = torch.zeros(5, dtype=torch.int64)


def test_backend_refusals():
    be = hb.HipBackend()
    cache = PagedKVCache(config(), 3, "cpu", FP4)
    kc, vc, scales = cache.k[0], cache.v[0], cache.scales(0)
    q, k = torch.zeros(5, 4, 128, dtype=torch.bfloat16), torch.zeros(5, 2, 128, dtype=torch.bfloat16)
    cos = torch.zeros(5, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="4-bit pool, q, k and v"):
        be.forward(q.float(), k.float(), k.float(), kc, vc, Meta, **scales)
    with pytest.raises(ValueError, match="4-bit pool, q, k and v"):
        be.forward(q, k.half(), k, kc, vc, Meta, **scales)
    with pytest.raises(ValueError, match="block scales"):
        be.forward(q, k, k, kc, vc, Meta)
    with pytest.raises(ValueError, match="block scales"):
        be.forward_rotary(q, k, k, cos, cos, kc, vc, Meta, k_scale=0.5, v_scale=0.5)
    with pytest.raises(ValueError, match="Hkv, Dh"):
        be.forward(q[..., :64], k[..., :64], k[..., :64], kc, vc, Meta, **scales)
    with pytest.raises(ValueError, match="block size"):
        be.forward(q, k, k, PagedKVCache(config(), 3, "cpu", FP4, 32).k[0], PagedKVCache(config(), 3, "cpu", FP4, 32).v[0],
                   Meta, **scales)
    with pytest.raises(ValueError, match="of one dtype"):
        be.append(k[..., :64], k[..., :64], kc, vc, Meta, **scales)
    with pytest.raises(ValueError, match="describe k's tokens"):
        be.append(k[:3], k[:3], kc, vc, Meta, **scales)
    with pytest.raises(ValueError, match="block scales"):
        be.append(k, k, kc, vc, Meta)
    with pytest.raises(ValueError, match="block scales"):
        be.attend(q, kc, vc, Meta, q)
    for kw, match in ((dict(q=q[:3]), "N, H, Dh"), (dict(q=q[:, :3]), "N, H, Dh"), (dict(q=q[..., :64]), "N, H, Dh"),
                      (dict(out=q.float()), "out must be like q"), (dict(out=q[:, :2]), "out must be like q"),
                      (dict(out=torch.zeros(5, 4, 256, dtype=q.dtype)[..., ::2]), "unit stride"), (dict(vc=vc[:2]), "alike"),
                      (dict(out=q.to("meta")), "one device"), (dict(q=q.to("meta")), "one device")):
        a = dict(q=q, vc=vc, out=torch.empty_like(q)) | kw
        with pytest.raises(ValueError, match=match):
            be.attend(a["q"], kc, a["vc"], Meta, a["out"], **scales)
    with pytest.raises(ValueError, match="one device"):
        be.append(k, k.to("meta"), kc, vc, Meta, **scales)
    with pytest.raises(ValueError, match="one device"):
        be.forward(q.to("meta"), k, k, kc, vc, Meta, **scales)
    # 16-bit pools take neither
    p16 = torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="fp8 pools only"):
        be.forward(q, k, k, p16, p16.clone(), Meta, **scales)
    w = torch.ones(128, dtype=torch.bfloat16)
    for bad in ((w[:64], w, 1e-5), (w, w.float(), 1e-5), (w, torch.ones(256, dtype=torch.bfloat16)[::2], 1e-5)):
        with pytest.raises(ValueError, match="weights must be contiguous"):
            be.rope_append(q, k, k, cos, cos, p16, p16.clone(), Meta, qk_norm=bad)
    for bad_k, bad_v in ((k.float(), k), (k, k.half()), (k.to("meta"), k)):
        for call in (be.rope_append, be.forward_rotary):
            with pytest.raises(ValueError, match="with head norms, q, k and v"):
                call(q, bad_k, bad_v, cos, cos, p16, p16.clone(), Meta, qk_norm=(w, w, 1e-5))
    for eps in (-1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="eps"):
            be.forward_rotary(q, k, k, cos, cos, p16, p16.clone(), Meta, qk_norm=(w, w, eps))
    with pytest.raises(ValueError, match="cos and sin"):
        be.rope_append(q, k, k, cos[:3], cos[:3], p16, p16.clone(), Meta, qk_norm=(w, w, 1e-5))


def test_qk_norm_rope_refusals():
    from minillm.model import kernels

    q, k = torch.zeros(1, 4, 5, 128, dtype=torch.bfloat16), torch.zeros(1, 2, 5, 128, dtype=torch.bfloat16)
    cos, w = torch.zeros(1, 5, 128, dtype=torch.bfloat16), torch.ones(128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="match q"):
        kernels.qk_norm_rope(q, k[:, :, :3], cos, cos, w, w, 1e-5)
    with pytest.raises(ValueError, match="cos and sin must be"):
        kernels.qk_norm_rope(q, k, cos[:, :4], cos, w, w, 1e-5)
    with pytest.raises(ValueError, match="one dtype"):
        kernels.qk_norm_rope(q, k.half(), cos, cos, w, w, 1e-5)
    with pytest.raises(ValueError, match="on a GPU"):
        kernels.qk_norm_rope(q, k, cos, cos, w, w, 1e-5)
    assert not kernels.qk_norm_rope_ok(q[..., :120], k[..., :120], cos[..., :120], cos[..., :120])  # Dh % 16
    assert not kernels.qk_norm_rope_ok(q[..., 4:116], k[..., 4:116], cos[..., :112], cos[..., :112])  # not 16-byte aligned
    assert kernels.qk_norm_rope_ok(q, k, cos, cos)


def test_entry_points_check_their_arguments():
    lib = _native.lib()
    a = 1 << 20  # an aligned address that nothing reads: every call below is refused before its launch
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        lib.call("mllm_kv_append_fp4", a, 256, 128, a, 256, 128, 0, a, a, a, a, 4, 16, 2, 128, a, 1, None)
    with pytest.raises(ValueError, match="multiple of 32"):
        lib.call("mllm_kv_append_fp4", a, 256, 80, a, 256, 80, 2, a, a, a, a, 4, 16, 2, 80, a, 1, None)
    with pytest.raises(ValueError, match="16-byte aligned"):
        lib.call("mllm_kv_append_fp4", a + 2, 256, 128, a, 256, 128, 2, a, a, a, a, 4, 16, 2, 128, a, 1, None)
    with pytest.raises(ValueError, match="16-byte aligned"):
        lib.call("mllm_kv_append_fp4", a, 257, 128, a, 256, 128, 2, a, a, a, a, 4, 16, 2, 128, a, 1, None)
    with pytest.raises(ValueError, match="null pointer"):
        lib.call("mllm_kv_append_fp4", a, 256, 128, a, 256, 128, 2, a, a, None, a, 4, 16, 2, 128, a, 1, None)
    with pytest.raises(ValueError, match="too many tokens"):
        lib.call("mllm_kv_append_fp4", a, 256, 128, a, 256, 128, 2, a, a, a, a, 4, 16, 2, 128, a, 1 << 40, None)
    with pytest.raises(ValueError, match="null pointer"):
        lib.call("mllm_kv_read_fp4", a, a, a, a, 4, 16, 2, 128, a, 1, 2, a, None, None)
    lib.call("mllm_kv_append_fp4", None, 0, 0, None, 0, 0, 2, None, None, None, None, 0, 16, 2, 128, None, 0, None)
    lib.call("mllm_kv_read_fp4", None, None, None, None, 0, 16, 2, 128, None, 0, 2, None, None, None)

    def decode(h=32, hkv=8, dh=128, bs=16, split=8, dtype=2, ws=0, merges=0, q=a, scales=a):
        lib.call("mllm_paged_decode_fp4", q, 4096, 128, a, a, scales, a, 4, bs, h, hkv, dh, a, a, a, 10, a, merges, split, 0.1, dtype,
                 a, 4096, 128, None, ws, None)

    for kw, match in ((dict(dh=64), "head_dim"), (dict(bs=24), "block_size"), (dict(h=30), "multiple of num_kv_heads"),
                      (dict(h=17, hkv=1), "at most 16"), (dict(split=193), "pages_per_split"), (dict(dtype=0), "dtype"),
                      (dict(merges=1), "workspace"), (dict(q=a + 8), "aligned"), (dict(scales=None), "null pointer"),
                      (dict(bs=1 << 26), "too large")):
        with pytest.raises(ValueError, match=match):
            decode(**kw)
    with pytest.raises(ValueError, match="null pointer"):
        lib.call("mllm_paged_prefill_fp4", a, 4096, 128, a, a, None, a, 4, 16, 32, 8, 128, a, a, a, a, a, 1, 32, 0.1, 2, a, 4096,
                 128, None)

    def norm(q_norm=a, k_norm=a, eps=1e-5, **kw):
        args = _native.RopeAppend(**{**dict(
            q=a, k=a, v=a, q_stride_tok=512, q_stride_head=128, k_stride_tok=256, k_stride_head=128, v_stride_tok=256,
            v_stride_head=128, cos=a, sin=a, cs_stride_tok=128, q_out=a, q_out_stride_tok=512, q_out_stride_head=128,
            k_cache=a, v_cache=a, k_scales=a, v_scales=a, k_scale=1.0, v_scale=1.0, num_blocks=4, slot_mapping=a,
            num_tokens=1, block_size=16, num_heads=4, num_kv_heads=2, head_dim=128, dtype=2, pool=2), **kw})
        lib.call("mllm_qk_norm_rope_kv_append", ctypes.addressof(args), q_norm, k_norm, eps, None)

    for kw, match in ((dict(q_norm=None), "go together"), (dict(q_norm=None, k_norm=None, pool=0), "4-bit pools only"),
                      (dict(pool=3), "unknown pool"), (dict(head_dim=96), "multiple of 64"), (dict(head_dim=120, pool=0), "multiple of 16"),
                      (dict(head_dim=1040, pool=0), "at most 1024"), (dict(eps=-1.0), "eps"), (dict(dtype=0), "dtype"),
                      (dict(k_scales=None), "null pointer"), (dict(q=a + 2), "aligned"), (dict(k_stride_tok=129), "aligned"),
                      (dict(pool=1, k_scale=0.0), "positive"), (dict(num_tokens=-1), "sizes"),
                      (dict(num_tokens=(1 << 31) - 1, num_heads=64), "too many")):
        with pytest.raises(ValueError, match=match):
            norm(**kw)
    norm(num_tokens=0, q=None)
    with pytest.raises(ValueError, match="null arguments"):
        lib.call("mllm_qk_norm_rope_kv_append", None, a, a, 1e-5, None)
    with pytest.raises(ValueError, match="null pointer"):
        lib.call("mllm_qk_norm_rope", a, 512, 128, 128, a, 512, 128, 128, a, a, 128, 128, a, None, 1e-5, 1, 1, 4, 2, 128, 2, a, a, None)


def test_layer_pool_checks():
    lib = _native.lib()
    fwd = lib.fn("mllm_attention_forward_pool")
    step = _native.LayerStep(num_heads=32, num_kv_heads=8, head_dim=128, block_size=16, dtype=2, softmax_scale=0.1)
    at = ctypes.addressof(step)

    def call(pool, cos=None, sin=None, q_rot=None):
        lib.check(fwd(at, 0, 0, 0, 0, 0, 0, 0, 0, 0, cos, sin, 0, q_rot, None if pool is None else ctypes.addressof(pool), 0, None))

    ones = dict(k_scale=1.0, v_scale=1.0)
    with pytest.raises(ValueError, match="null pool"):
        call(None)
    with pytest.raises(ValueError, match="go together"):
        call(_native.LayerPool(q_norm=1 << 20, **ones))
    with pytest.raises(ValueError, match="with cos and sin"):
        call(_native.LayerPool(q_norm=1 << 20, k_norm=1 << 20, **ones))
    step.kv_fp8 = 2
    with pytest.raises(ValueError, match="fp8 pools only"):
        call(_native.LayerPool(k_scale=0.5, v_scale=1.0))
    call(_native.LayerPool(**ones))  # no tokens and no work
    # without k, v and cos the attention alone, here of no rows; a missing k or v, or none in the older call, is refused
    step.num_tokens = 3
    call(_native.LayerPool(**ones))
    some, pool = 1 << 20, _native.LayerPool(**ones)
    for k, v in ((some, None), (None, some)):
        with pytest.raises(ValueError, match="null pointer"):
            lib.check(fwd(at, some, 0, 0, k, 0, 0, v, 0, 0, None, None, 0, None, ctypes.addressof(pool), some, None))
    step.kv_fp8 = 0
    with pytest.raises(ValueError, match="null pointer"):
        lib.call("mllm_attention_forward", at, some, 0, 0, None, 0, 0, None, 0, 0, None, None, 0, None, some, some, 1.0, 1.0, some, None)
    step.kv_fp8, step.num_tokens = 3, 0
    with pytest.raises(ValueError, match="unknown pool"):
        call(_native.LayerPool(**ones))


@pytest.mark.parametrize("name", ["RopeAppend", "LayerPool"])
def test_structs_match_the_header(tmp_path, name):
    import subprocess
    from pathlib import Path

    cls = getattr(_native, name)
    c_name = {"RopeAppend": "mllm_rope_append", "LayerPool": "mllm_layer_pool"}[name]
    fields = [f for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "minillm_hip.h"\nint main(void) {\n'
                   f'printf("%zu\\n", sizeof({c_name}));\n'
                   + "".join(f'printf("%zu\\n", offsetof({c_name}, {f}));\n' for f in fields) + "return 0;\n}\n")
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", "-std=c99", f"-I{include}", str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def test_config_names_head_norms():
    d = {k: v for k, v in LLAMA_3_1_8B.items()}
    assert LlamaConfig.from_dict(d).qk_norm is False
    assert LlamaConfig.from_dict({**d, "qk_norm": True}).qk_norm is True


class Recorder:
    """A library that launches nothing and keeps what `mllm_attention_forward_pool` was asked for."""

    def __init__(self):
        self.steps, self.plans = [], 0

    def call(self, name, *args):
        self.plans += name == "mllm_plan"

    def launch(self, device, name, *args):
        assert name == "mllm_attention_forward_pool"
        step = _native.LayerStep.from_address(args[0])
        self.steps.append({f: getattr(step, f) for f, _ in step._fields_})

    def workspace_bytes(self, num_work, num_heads, head_dim):
        return 4 * num_work * num_heads * head_dim


def test_head_counts_are_each_calls_own(monkeypatch):
    # one step's metadata with layers of other head counts: the plan and the step's arguments follow the call
    from minillm.attention.metadata import AttentionMetadata

    monkeypatch.setattr(_native, "stream_ptr", lambda device: 0)
    be = hb.HipBackend()
    be._lib, be.check_plan = Recorder(), False
    meta = AttentionMetadata._arenas(16, [0, 1, 2, 22], [300, 40, 20], 22, 19, 24, "cpu")
    layouts = [(32, 8), (8, 8), (8, 2), (32, 8), (2, 2)]
    for h, hkv in layouts:
        cache = PagedKVCache(config(num_attention_heads=h, num_key_value_heads=hkv), 24, "cpu", FP4)
        q = torch.zeros(22, h, 128, dtype=torch.bfloat16)
        for _ in range(2):  # the second call finds the first one's
            be.attend(q, cache.k[0], cache.v[0], meta, torch.empty_like(q), **cache.scales(0))
    assert be._lib.plans == len(layouts)
    for i, (h, hkv) in enumerate(layouts):
        a, b = be._lib.steps[2 * i:2 * i + 2]
        assert a == b and (a["num_heads"], a["num_kv_heads"], a["head_dim"]) == (h, hkv, 128)
        assert a["q_tile_tokens"] == hb.prefill_q_tile([1, 1, 20], h // hkv, hkv) and a["kv_fp8"] == 2
        assert a["pages_per_split"] == hb.pages_per_split(22, hkv, h, kv_fp4=True)
        assert a["workspace_bytes"] == 4 * a["num_decode_work"] * h * 128 > 0
    # the other pools' layers
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        for h, hkv, dh in ((32, 8, 128), (8, 8, 128), (8, 2, 128), (8, 2, 64)):
            pool = torch.zeros(24, 16, hkv, dh, dtype=torch.uint8 if dtype.itemsize == 1 else dtype).view(dtype)
            for _ in range(2):
                step = _native.LayerStep.from_address(be.layer_step(meta, 22, h, torch.bfloat16, pool))
                assert (step.num_heads, step.num_kv_heads, step.head_dim) == (h, hkv, dh)
                assert step.workspace_bytes == 4 * step.num_decode_work * h * dh
    assert be._lib.plans == len(layouts) + 8


def test_a_16bit_pool_takes_a_scale_of_one_as_a_tensor():
    be = hb.HipBackend()
    p16 = torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16)
    q, k = torch.zeros(5, 4, 128, dtype=torch.bfloat16), torch.zeros(5, 2, 128, dtype=torch.bfloat16)
    for one in (1.0, 1, torch.tensor(1.0), torch.ones(1, dtype=torch.float64)):
        assert len(be._check(q, k, k, p16, p16.clone(), Meta, one, one)) == 3
    for bad in (0.5, torch.tensor(0.5), torch.ones(2), torch.tensor([127], dtype=torch.uint8).view(E8M0)):
        for scales in ((1.0, bad), (bad, 1.0)):
            with pytest.raises(ValueError, match="fp8 pools only"):
                be._check(q, k, k, p16, p16.clone(), Meta, *scales)


def test_tables_and_pools_of_another_device_are_refused():
    be = hb.HipBackend()
    w = torch.ones(128, dtype=torch.bfloat16)
    q, k = torch.zeros(5, 4, 128, dtype=torch.bfloat16), torch.zeros(5, 2, 128, dtype=torch.bfloat16)
    cos = torch.zeros(5, 128, dtype=torch.bfloat16)
    cache, p16 = PagedKVCache(config(), 3, "cpu", FP4), torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16)
    pools = {"norms": (p16, p16.clone(), dict(qk_norm=(w, w, 1e-5))), "fp4": (cache.k[0], cache.v[0], cache.scales(0)),
             "both": (cache.k[0], cache.v[0], dict(qk_norm=(w, w, 1e-5), **cache.scales(0)))}
    for kc, vc, kw in pools.values():
        for call in (be.rope_append, be.forward_rotary):
            for c, s in ((cos.to("meta"), cos), (cos, cos.to("meta"))):
                with pytest.raises(ValueError, match="one device"):
                    call(q, k, k, c, s, kc, vc, Meta, **kw)
            for a, b in ((kc.to("meta"), vc), (kc, vc.to("meta"))):
                with pytest.raises(ValueError, match="one device|pool's device"):
                    call(q, k, k, cos, cos, a, b, Meta, **kw)


def test_a_plan_is_launched_with_its_device_current(monkeypatch):
    # as the launches behind it are (NativeLib.launch); two devices that are only named
    be, current, seen = hb.HipBackend(), [0], []

    class On:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(_native, "stream_ptr", lambda device: 100 + device.index)
    monkeypatch.setattr(be, "_make_plan", lambda meta, h, hkv, dh, device, stream, pool: seen.append((current[0], stream)))
    be.plan(Meta, 32, 8, 128, torch.device("cuda:0"), pool=2)
    be.plan(Meta, 32, 8, 128, torch.device("cuda:1"), pool=2)
    assert seen == [(0, 100), (1, 101)] and current == [0]
