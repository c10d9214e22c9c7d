"""A decoder layer served from reduced storage, its operators together as the engine runs them: projections of 8-bit blocks,
norms of q and k with the rotation and the 4-bit append, attention over the 4-bit pool.

- one host call per layer gives the bits of the kernels called one by one, every replay of a captured step those of the eager
  step;
- a layer's attention against float64 from the formulas, over the pool's values;
- the engine (chunked prompts, shared prompt heads, preemption, graphs) against itself with attention in float64 over the same
  pool's values.  These runs have one layer, whose q, k, v come from 8-bit blocks and whose other products are 16-bit: a
  token's k and v then depend on nothing but the token and its place, and no later rounding to few bits can turn a
  difference in the last bit of an attention output into a larger one, so tokens are compared as on a 16-bit pool.
"""

import math

import pytest
import torch

from harness import bits
from naive import causal_allowed
from test_gpu_engine import assert_greedy_match, prompts, run_engine

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP4 = torch.float4_e2m1fn_x2
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], dtype=torch.float64)


def make_model(seed, layers=2, heads=4, kv_heads=2, dtype=torch.bfloat16, norms=True):
    from minillm.model.config import LlamaConfig
    from minillm.model.llama import LlamaForCausalLM, random_init_

    cfg = LlamaConfig(vocab_size=256, hidden_size=heads * 128, intermediate_size=1024, num_hidden_layers=layers,
                      num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=128, rms_norm_eps=1e-5,
                      rope_theta=10000.0, max_position_embeddings=4096, qk_norm=norms)
    model = random_init_(LlamaForCausalLM(cfg).to(device=DEV, dtype=dtype), std=0.05, seed=seed)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        model.lm_head.weight.mul_(12)
        for layer in model.model.layers if norms else ():
            for norm in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                norm.weight.copy_(torch.rand(128, generator=g) + 0.5)
    return model


def pool_values(codes, scales):
    """A pool's codes [nb, bs, Hkv, Dh / 2] and scales with the same leading places -> float64 [nb, bs, Hkv, Dh]."""
    c = codes.view(torch.uint8).long()
    values = GRID.to(c.device)[torch.stack((c & 15, c >> 4), dim=-1).flatten(-2)]
    return values * torch.exp2(scales.view(torch.uint8).double() - 127).repeat_interleave(32, -1)


class PlainAttention:
    """The kernels' append (with norms and rotation), attention in float64 over the pool's values."""

    name = "plain"
    fuse_rotary = True

    def __init__(self):
        from minillm.attention import get_backend

        self.hip = get_backend("hip")

    def forward_rotary(self, q, k, v, cos, sin, k_cache, v_cache, meta, k_scale=1.0, v_scale=1.0, qk_norm=None):
        q = self.hip.rope_append(q, k, v, cos, sin, k_cache, v_cache, meta, k_scale, v_scale, qk_norm=qk_norm)
        nb, bs, hkv, _ = k_cache.shape
        kd = pool_values(k_cache, k_scale.permute(0, 1, 3, 2)).flatten(0, 1)
        vd = pool_values(v_cache, v_scale.permute(0, 3, 1, 2)).flatten(0, 1)
        out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
        indptr, indices = meta.kv_indptr.tolist(), meta.kv_indices
        for i, (at, end, length) in enumerate(zip(meta.query_start_loc, meta.query_start_loc[1:], meta.seq_lens)):
            n = end - at
            pages = indices[indptr[i]:indptr[i + 1]].long()
            slots = (pages[:, None] * bs + torch.arange(bs, device=q.device)).flatten()[:length]
            blocked = ~causal_allowed(n, length).to(q.device)
            for h in range(q.shape[1]):
                x = h // (q.shape[1] // hkv)
                s = q[at:at + n, h].double() @ kd[slots, x].t().contiguous() / math.sqrt(128)
                out[at:at + n, h] = torch.softmax(s.masked_fill(blocked, -math.inf), -1) @ vd[slots, x]
        return out.to(q.dtype)


KW = dict(max_batch_size=8, num_kv_blocks=300, max_model_len=2048, kv_cache_dtype=FP4)


@pytest.mark.parametrize("pool", ["16bit", "fp8", "fp4"])
@pytest.mark.parametrize("norms", [True, False])
def test_one_call_layer_equals_the_kernels_one_by_one(hip, monkeypatch, pool, norms):
    from minillm.attention import get_backend
    from minillm.model import kernels

    model = make_model(seed=3, norms=norms)
    kw = dict(KW, kv_cache_dtype={"16bit": torch.bfloat16, "fp8": torch.float8_e4m3fn, "fp4": FP4}[pool])
    if pool == "fp8":
        kw["kv_scales"] = (0.5, 0.25)
    ps, whole, calls = prompts(6, 1, 150, seed=4), kernels.decoder_layer, []

    def counted(*args):
        out = whole(*args)
        calls.append(out is not None)
        return out

    monkeypatch.setattr(kernels, "decoder_layer", counted)
    one_call, _ = run_engine(model, get_backend("hip"), None, ps, 12, **kw)
    assert any(calls)
    monkeypatch.setattr(kernels, "decoder_layer", lambda *args: None)
    separate, _ = run_engine(model, get_backend("hip"), None, ps, 12, **kw)
    assert one_call == separate  # tokens and the margins of the logits


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("blocks8", [True, False])
def test_every_replay_equals_the_eager_step(hip, dtype, blocks8):
    # prompts (eager) and replays of other buckets in between, as the batch fills and drains
    from minillm.attention import get_backend
    from minillm.engine.core import AddRequest, EngineCore
    from minillm.model.fp8 import quantize_

    model = make_model(seed=31, dtype=dtype)
    if blocks8:
        quantize_(model)
    model.set_backend(get_backend("hip"))
    core = EngineCore(model, decode_graphs=(2, 8), **KW)
    for i, (p, n) in enumerate(zip(prompts(5, 1, 700, seed=32), (4, 7, 9, 30, 40))):
        core.add_request(AddRequest(f"r{i}", p, n, ignore_eos=True))
    seen, buckets = 0, set()
    while core.has_work():
        core.step()
        if core.graphs.replays == seen:
            continue
        seen = core.graphs.replays
        c = core.graphs._captured[core.graphs.last_bucket]
        got_logits, got_tokens = c.logits.clone(), c.tokens.clone()
        ref_logits, ref_tokens = core.graphs.eager_reference()
        torch.cuda.synchronize()
        assert torch.equal(got_tokens, ref_tokens), core.graphs.last_bucket
        assert torch.equal(got_logits.view(torch.int16), ref_logits.view(torch.int16)), core.graphs.last_bucket
        assert torch.isfinite(got_logits).all()
        buckets.add(core.graphs.last_bucket)
    assert seen >= 30 and buckets == {2, 8}


@pytest.mark.parametrize("steps", [
    [(37, 1), (128, 1), (211, 1), (500, 1)], [(17 * i % 300, 1) for i in range(40)], [(90, 1), (0, 30), (250, 1), (7, 5)],
    [(2000, 1), (3, 1), (9000, 1)], [(5, 1)]], ids=["4_rows", "40_rows", "mixed", "long", "one"])
@pytest.mark.parametrize("h,hkv", [(32, 8), (4, 2)])
def test_a_step_is_the_same_bits_by_every_route(hip, steps, h, hkv):
    # one call per layer, separate launches, prefill on a second stream, and (decode steps) the staged metadata of a
    # captured graph whose bucket the step fills
    from minillm.attention.hip_backend import HipBackend, device_cus, pages_per_split
    from minillm.attention.metadata import AttentionMetadata, DeviceBlockTables, SeqStep, StaticDecodeMetadata
    from test_gpu_fp4 import append, make_cache

    g = torch.Generator().manual_seed(71)
    need = [-(-(c + n) // 16) for c, n in steps]
    ids = torch.randperm(sum(need) + 4, generator=g).tolist()
    seqs = [SeqStep(c, n, [ids.pop() for _ in range(w)]) for (c, n), w in zip(steps, need)]
    total = (sum(need) + 4) * 16
    past = [torch.randn(total, hkv, 128, generator=g).bfloat16().to(DEV) for _ in range(2)]
    k, v = (torch.randn(sum(n for _, n in steps), hkv, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    q = torch.randn(k.shape[0], h, 128, generator=g).bfloat16().to(DEV)
    results = {}
    for route in ("one_call", "separate", "second_stream", "staged"):
        be, cache = HipBackend(), make_cache(hkv, sum(need) + 4)
        append(cache, *past, torch.arange(total, device=DEV))
        pools = cache.k[0], cache.v[0]
        if route == "staged":
            if any(n > 1 for _, n in steps):
                continue
            static = StaticDecodeMetadata(len(seqs), DeviceBlockTables(len(seqs), sum(need), DEV), 16)
            static.load(list(range(len(seqs))), seqs,
                        pages_per_split(sum(need), hkv, h, False, device_cus(DEV), kv_fp4=True))
            static.build()
            meta = static.meta
        else:
            meta = AttentionMetadata.build(seqs, 16, DEV)
        if route in ("separate", "staged"):
            out = torch.empty_like(q)
            be.append(k, v, *pools, meta, **cache.scales(0))
            be.attend(q, *pools, meta, out, **cache.scales(0))
        else:
            be.overlap_mixed = route == "second_stream"
            out = be.forward(q, k, v, *pools, meta, **cache.scales(0))
        torch.cuda.synchronize()
        results[route] = out
    for route, out in results.items():
        assert torch.equal(bits(out), bits(results["one_call"])), route


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_against_float64(hip, dtype):
    # LlamaAttention on a mixed paged step: q and k normed and rotated by the formula from the layer's own projections, over the
    # pool's values.  On top of the attention's own error (test_gpu_fp4) q is rounded once, half a step: a score moves by
    # at most eps / 2 of sum_d |q_d k_d| / sqrt(Dh), twice that in a weight's logarithm.
    from test_gpu_qk_norm import formula

    from minillm.attention.metadata import AttentionMetadata, SeqStep
    from minillm.cache.paged import PagedKVCache, PagedStep
    from minillm.model.fp8 import quantize_

    model = quantize_(make_model(seed=5, layers=1, heads=8, kv_heads=2, dtype=dtype))
    attn, cache = model.model.layers[0].self_attn, PagedKVCache(model.config, 30, DEV, FP4)
    g = torch.Generator().manual_seed(6)
    eps, lengths = torch.finfo(dtype).eps, [0, 0, 0]
    tables = [[7, 2, 29, 11, 3, 8, 4, 1, 6], [5], [0, 9, 10]]
    for new in ((130, 1, 17), (1, 1, 20), (1, 1, 1)):
        n = sum(new)
        meta = AttentionMetadata.build([SeqStep(c, m, t) for c, m, t in zip(lengths, new, tables)], 16, DEV)
        positions = torch.cat([torch.arange(c, c + m) for c, m in zip(lengths, new)])[None].to(DEV)
        lengths = [c + m for c, m in zip(lengths, new)]
        x = torch.randn(1, n, 1024, generator=g).to(dtype).to(DEV)
        cos, sin = model.model.rotary_emb(positions, dtype)
        with torch.no_grad():
            got = attn.attend(x, cos, sin, PagedStep(cache, meta)).view(n, 8, 128).double()
            q = attn.q_proj(x).view(1, n, 8, 128).transpose(1, 2)
        q = formula(q, attn.q_norm.weight, cos, sin, 1e-5)[0][0]
        at = 0
        for m, length, table in zip(new, lengths, tables):
            slots = torch.tensor([table[p // 16] * 16 + p % 16 for p in range(length)], device=DEV)
            kd, vd = (t.double() for t in cache.read(0, slots, dtype))
            blocked = ~causal_allowed(m, length).to(DEV)
            for head in range(8):
                kk, vv, qq = kd[:, head // 4].contiguous(), vd[:, head // 4].contiguous(), q[head, at:at + m]
                p = torch.softmax((qq @ kk.t().contiguous() / math.sqrt(128)).masked_fill(blocked, -math.inf), -1)
                o, a = p @ vv, p @ vv.abs()
                size = (qq.abs() @ kk.abs().t().contiguous() / math.sqrt(128)).masked_fill(blocked, 0).amax(-1)
                ds = (eps / 2 * 1.01 + 140 * 2.0 ** -24) * size  # q's 1%: its rounding relative to the formula's q, and fp32 norms
                bound = eps / 2 * o.abs() + (eps / 2 + 2 * ds[:, None] + 2.0 ** -20) * a
                worst = ((got[at:at + m, head] - o).abs() / bound.clamp_min(1e-30)).max().item()  # v of 0: both 0
                assert worst <= 1, f"length {length} head {head}: {worst:.3f} of its bound"
            at += m


def one_layer(seed, dtype):
    from minillm.model.fp8 import Fp8Linear

    model = make_model(seed, layers=1, dtype=dtype)
    attn = model.model.layers[0].self_attn
    for name in ("q_proj", "k_proj", "v_proj"):
        setattr(attn, name, Fp8Linear.from_linear(getattr(attn, name)))
    return model


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_engine_matches_plain_attention(hip, dtype):
    from minillm.attention import get_backend
    from minillm.attention.metadata import AttentionMetadata

    model = one_layer(41, dtype)
    ps = prompts(10, 1, 300, seed=42)
    exp, _ = run_engine(model, PlainAttention(), AttentionMetadata.build, ps, 20, **KW)
    got, core = run_engine(model, get_backend("hip"), None, ps, 20, decode_graphs=True, **KW)
    assert_greedy_match(got, exp)
    assert core.cache.k[0].dtype == FP4 and core.graphs.replays > 10
    chunked, core = run_engine(model, get_backend("hip"), None, ps, 20, chunked_prefill=True, max_num_batched_tokens=96,
                               step_log=True, **KW)
    assert_greedy_match(chunked, exp)
    assert any(r.prefill_tokens and r.decode_tokens for r in core.step_log)


def test_engine_with_preemption_and_prefix_sharing(hip):
    from minillm.attention import get_backend
    from minillm.attention.metadata import AttentionMetadata

    model = one_layer(43, torch.float16)
    head = prompts(1, 48, 49, seed=5)[0]
    ps = [head + p for p in prompts(6, 5, 40, seed=6)]
    exp, _ = run_engine(model, PlainAttention(), AttentionMetadata.build, ps, 40, **KW)
    got, core = run_engine(model, get_backend("hip"), None, ps, 40, decode_graphs=True,
                           **dict(KW, num_kv_blocks=24, max_batch_size=6))
    assert_greedy_match(got, exp)
    st = core.stats()
    assert st.num_preemptions > 0 and st.prefix_cache_hits > 0


@pytest.mark.parametrize("t", [1, 40, 300])
def test_contiguous_model_of_the_same_weights(hip, t):
    # without a cache (q and k normed and rotated in one launch): the same as with the modules' own norms and rotation, within
    # their 16-bit roundings: the fused one rounds once, the modules three times (norm, weight, rotation)
    from minillm.model import kernels
    from minillm.model.fp8 import quantize_

    model = quantize_(make_model(seed=8, layers=1))
    attn = model.model.layers[0].self_attn
    x = torch.randn(2, t, 512, generator=torch.Generator().manual_seed(t)).bfloat16().to(DEV)
    cos, sin = model.model.rotary_emb(torch.arange(t, device=DEV).expand(2, t), torch.bfloat16)
    with torch.no_grad():
        q, k, v = (p(x).view(2, t, -1, 128).transpose(1, 2) for p in (attn.q_proj, attn.k_proj, attn.v_proj))
        assert kernels.qk_norm_rope_ok(q, k, cos, sin)
        got = attn.attend(x, cos, sin)
        want = attn._contiguous(*kernels.qk_norm_rope(q, k, cos, sin, attn.q_norm.weight, attn.k_norm.weight, 1e-5), v, None)
    assert torch.equal(bits(got), bits(want))


def test_two_steps_on_two_streams(hip):
    # appends and attention of two steps over two layers' pools, each on its own stream with its own backend, at once
    from test_gpu_fp4 import append, make_cache

    from minillm.attention import get_backend
    from minillm.attention.metadata import AttentionMetadata, SeqStep

    g = torch.Generator().manual_seed(9)
    jobs = []
    for rows in ([(3000, 1), (70, 1), (900, 1)], [(64, 200), (1500, 1), (0, 33)]):
        need = [-(-(c + n) // 16) for c, n in rows]
        ids = torch.randperm(sum(need), generator=g).tolist()
        meta = AttentionMetadata.build([SeqStep(c, n, [ids.pop() for _ in range(w)]) for (c, n), w in zip(rows, need)], 16, DEV)
        cache = make_cache(8, sum(need))
        append(cache, *(torch.randn(16 * sum(need), 8, 128, generator=g).bfloat16().to(DEV) for _ in range(2)),
               torch.arange(16 * sum(need), device=DEV))
        n = sum(m for _, m in rows)
        q, k, v = (torch.randn(n, h, 128, generator=g).bfloat16().to(DEV) for h in (32, 8, 8))
        be = get_backend("hip")
        jobs.append((be, (q, k, v, cache.k[0], cache.v[0], meta), cache.scales(0), be.forward(q, k, v, cache.k[0], cache.v[0], meta,
                                                                                           **cache.scales(0))))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in jobs], [[], []]
    for _ in range(5):
        for (be, args, scales, _), s, out in zip(jobs, streams, got):
            with torch.cuda.stream(s):
                out.append(be.forward(*args, **scales))
    torch.cuda.synchronize()
    for (*_, want), outs in zip(jobs, got):
        assert all(torch.equal(bits(o), bits(want)) for o in outs)


@pytest.mark.parametrize("paged", [True, False])
def test_other_norms_are_called_as_they_are(hip, monkeypatch, paged):
    # norms of another class, and hooked ones, keep their own forward; so does the whole layer around them
    from minillm.attention import get_backend
    from minillm.attention.metadata import AttentionMetadata, SeqStep
    from minillm.cache.paged import PagedKVCache, PagedStep
    from minillm.model import kernels

    def layer_norms(attn):
        for name in ("q_norm", "k_norm"):
            setattr(attn, name, torch.nn.LayerNorm(128, eps=1e-5, bias=False).to(DEV, torch.bfloat16))

    def hooked(attn):
        attn.k_norm.register_forward_hook(lambda m, args, out: 2 * out)

    n = 9
    x = torch.randn(1, n, 512, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    for change in (layer_norms, hooked):
        model = make_model(seed=8, layers=1)
        model.set_backend(get_backend("hip"))
        layer = model.model.layers[0]
        change(layer.self_attn)
        cos, sin = model.model.rotary_emb(torch.arange(n, device=DEV)[None], torch.bfloat16)
        results = []
        for fused in (True, False):
            with monkeypatch.context() as m:
                if not fused:
                    m.setattr(kernels, "head_norms_ok", lambda *args: False)
                cache = PagedKVCache(model.config, 2, DEV, FP4)
                step = PagedStep(cache, AttentionMetadata.build([SeqStep(0, n, [1])], 16, DEV)) if paged else None
                with torch.no_grad():
                    results.append(layer(x, cos, sin, step))
        assert torch.equal(bits(results[0]), bits(results[1])), change.__name__


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t", [1, 40, 300])
def test_contiguous_norms_and_rotation_against_the_modules(hip, monkeypatch, t, dtype):
    # What the attention of a model without a cache is given, against the formula and against the layer's own norm modules and
    # apply_rotary.  The fused launch rounds once: eps / 2 of the result, 2^-18 of the magnitudes it sums (test_gpu_qk_norm).  The
    # modules round the normed row, its product with the weight, the two products with cos and sin and their sum: with M
    # those magnitudes, at most 3 eps / 2 of M and eps / 2 of the result; 1% covers a rounding of a rounded value, and tiny
    # eps each rounding below the type's normal numbers.
    from test_gpu_qk_norm import formula

    from minillm.model import kernels
    from minillm.model.fp8 import quantize_
    from minillm.model.llama import apply_rotary

    model = quantize_(make_model(seed=8, layers=1, dtype=dtype))
    attn = model.model.layers[0].self_attn
    x = torch.randn(2, t, 512, generator=torch.Generator().manual_seed(t)) * torch.logspace(-3, 0, t)[:, None]  # eps counts
    x = x.to(dtype).to(DEV)
    cos, sin = model.model.rotary_emb(torch.arange(t, device=DEV).expand(2, t), dtype)
    given, fused, prefill, rotate = [], [], attn.backend.prefill, kernels.qk_norm_rope
    monkeypatch.setattr(attn.backend, "prefill", lambda *a, **kw: (given.append(a), prefill(*a, **kw))[1])
    monkeypatch.setattr(kernels, "qk_norm_rope", lambda *a: (fused.append(1), rotate(*a))[1])
    with torch.no_grad():
        out = attn.attend(x, cos, sin)
        q, k, v = (p(x).view(2, t, -1, 128).transpose(1, 2) for p in (attn.q_proj, attn.k_proj, attn.v_proj))
        own = [apply_rotary(norm(y), cos, sin) for norm, y in ((attn.q_norm, q), (attn.k_norm, k))]
    (got_q, got_k, got_v), = given
    assert fused == [1] and torch.equal(bits(got_v.contiguous()), bits(v.contiguous()))
    eps, tiny = torch.finfo(dtype).eps, torch.finfo(dtype).tiny
    for got, y, norm, other in ((got_q, q, attn.q_norm, own[0]), (got_k, k, attn.k_norm, own[1])):
        ref, mag = formula(y, norm.weight, cos, sin, 1e-5)
        once = eps / 2 * ref.abs() + 2.0 ** -18 * mag + tiny * eps
        assert bool(((got.double() - ref).abs() <= once).all())
        modules = 1.01 * (1.5 * eps * mag + eps / 2 * ref.abs()) + 2.0 ** -18 * mag + 8 * tiny * eps
        assert bool(((got.double() - other.double()).abs() <= once + modules).all())
    # and its result, against attention of them in float64: P and the output rounded, scores in fp32
    blocked = ~causal_allowed(t, t).to(DEV)
    for b in range(2):
        for head in range(4):
            qq, kk, vv = got_q[b, head].double(), got_k[b, head // 2].double().contiguous(), v[b, head // 2].double().contiguous()
            p = torch.softmax((qq @ kk.t().contiguous() / math.sqrt(128)).masked_fill(blocked, -math.inf), -1)
            o, a = p @ vv, p @ vv.abs()
            size = (qq.abs() @ kk.abs().t().contiguous() / math.sqrt(128)).masked_fill(blocked, 0).amax(-1, keepdim=True)
            bound = eps / 2 * o.abs() + (eps / 2 + 2 * 140 * 2.0 ** -24 * size + 2.0 ** -20) * a + tiny * eps
            assert bool(((out.view(2, t, 4, 128)[b, :, head].double() - o).abs() <= bound).all())
