"""The operators of long-lived sequences together, as the engine runs them: a model with rotary forms of long contexts served
from a pool of 8-bit blocks, requests that fork, a pool that is compacted between steps.

- a step is the same bits by every route (one host call per layer, separate launches, two streams, captured);
- the engine against itself with attention in float64 over the same pool's values;
- pages far into a pool larger than 32-bit offsets reach."""

import math
import random

import pytest
import torch

from harness import bits
from naive import causal_allowed
from test_gpu_engine import assert_greedy_match, prompts, run_engine

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP8 = torch.float8_e4m3fn
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 512}


def make_model(seed, layers=2, heads=4, kv_heads=2, dtype=torch.bfloat16, **kw):
    from minillm.model.config import LlamaConfig
    from minillm.model.llama import LlamaForCausalLM, random_init_

    cfg = LlamaConfig(vocab_size=256, hidden_size=heads * 128, intermediate_size=1024, num_hidden_layers=layers,
                      num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=128, rms_norm_eps=1e-5,
                      rope_theta=10000.0, max_position_embeddings=4096, **kw)
    model = random_init_(LlamaForCausalLM(cfg).to(device=DEV, dtype=dtype), std=0.05, seed=seed)
    with torch.no_grad():
        model.lm_head.weight.mul_(12)
    return model


KW = dict(max_batch_size=8, num_kv_blocks=300, max_model_len=2048, kv_cache_dtype=FP8, kv_scales="blocks")
FORMS = [{}, dict(rope_interleaved=True, rope_scaling=YARN, partial_rotary_factor=0.5), dict(qk_norm=True, rope_scaling=YARN)]


@pytest.mark.parametrize("steps", [
    [(37, 1), (128, 1), (211, 1), (500, 1)], [(17 * i % 300, 1) for i in range(40)], [(90, 1), (0, 30), (250, 1), (7, 5)],
    [(2000, 1), (3, 1), (9000, 1)], [(5, 1)]], ids=["4_rows", "40_rows", "mixed", "long", "one"])
@pytest.mark.parametrize("h,hkv", [(32, 8), (4, 2), (3, 1)])
def test_a_step_is_the_same_bits_by_every_route(hip, steps, h, hkv):
    from minillm.attention.hip_backend import HipBackend, device_cus, pages_per_split
    from minillm.attention.metadata import AttentionMetadata, DeviceBlockTables, SeqStep, StaticDecodeMetadata
    from test_gpu_fp8_blocks import append, make_cache

    if h == 3 and any(n > 1 for _, n in steps):
        pytest.skip("groups of three have no prefill kernel")
    g = torch.Generator().manual_seed(71)
    need = [-(-(c + n) // 16) for c, n in steps]
    ids = torch.randperm(sum(need) + 4, generator=g).tolist()
    seqs = [SeqStep(c, n, [ids.pop() for _ in range(w)]) for (c, n), w in zip(steps, need)]
    total = (sum(need) + 4) * 16
    past = [torch.randn(total, hkv, 128, generator=g).bfloat16().to(DEV) for _ in range(2)]
    k, v = (3 * torch.randn(sum(n for _, n in steps), hkv, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
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
        results[route] = [bits(out)] + [t.view(torch.uint8) for t in (*pools, cache.k_scale[0], cache.v_scale[0])]
    for route, got in results.items():
        assert all(torch.equal(a, b) for a, b in zip(got, results["one_call"])), route


@pytest.mark.parametrize("form", FORMS, ids=["reference", "yarn", "norms"])
def test_one_call_layer_equals_the_kernels_one_by_one(hip, monkeypatch, form):
    from minillm.attention import get_backend
    from minillm.model import kernels

    model = make_model(3, **form)
    ps, whole, calls = prompts(6, 1, 150, seed=4), kernels.decoder_layer, []

    def counted(*args):
        out = whole(*args)
        calls.append(out is not None)
        return out

    monkeypatch.setattr(kernels, "decoder_layer", counted)
    one_call, _ = run_engine(model, get_backend("hip"), None, ps, 12, **KW)
    assert any(calls) == ("rope_interleaved" not in form)  # a rotation by position goes layer by layer
    monkeypatch.setattr(kernels, "decoder_layer", lambda *args: None)
    separate, _ = run_engine(model, get_backend("hip"), None, ps, 12, **KW)
    assert one_call == separate  # tokens and the margins of the logits


@pytest.mark.parametrize("form", FORMS, ids=["reference", "yarn", "norms"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_replay_equals_the_eager_step(hip, dtype, form):
    from minillm.attention import get_backend
    from minillm.engine.core import AddRequest, EngineCore

    model = make_model(31, dtype=dtype, **form)
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


class PlainAttention:
    """The kernels' append (with rotation and norms where they go with it), attention in float64 over the pool's values."""

    name = "plain"
    fuse_rotary = True

    def __init__(self):
        from minillm.attention import get_backend

        self.hip = get_backend("hip")

    def forward_rotary(self, q, k, v, cos, sin, k_cache, v_cache, meta, k_scale=1.0, v_scale=1.0, qk_norm=None):
        q = self.hip.rope_append(q, k, v, cos, sin, k_cache, v_cache, meta, k_scale, v_scale, qk_norm=qk_norm)
        return self.attend(q, k_cache, v_cache, meta, k_scale, v_scale)

    def forward(self, q, k, v, k_cache, v_cache, meta, k_scale=1.0, v_scale=1.0):
        self.hip.append(k, v, k_cache, v_cache, meta, k_scale, v_scale)
        return self.attend(q, k_cache, v_cache, meta, k_scale, v_scale)

    def attend(self, q, k_cache, v_cache, meta, k_scale, v_scale):
        bs, hkv = k_cache.shape[1:3]
        kd, vd = ((c.double() * torch.exp2(s.view(torch.uint8).double() - 127)[:, None, :, None]).flatten(0, 1)
                  for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
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


@pytest.mark.parametrize("form", FORMS, ids=["reference", "yarn", "norms"])
@pytest.mark.parametrize("kw", [{}, dict(chunked_prefill=True, max_num_batched_tokens=64), dict(num_kv_blocks=45, max_model_len=600)],
                         ids=["plain", "chunked", "preempting"])
def test_engine_against_float64_attention(hip, form, kw):
    # one layer: a token's k and v depend on the token and its place alone, so both runs hold the same pool.  fp16 as on a
    # 16-bit pool, whose tokens are compared the same way
    from minillm.attention import get_backend

    model = make_model(13, layers=1, dtype=torch.float16, **form)
    ps = prompts(5, 20, 200, seed=14)
    ps.append(ps[2][:64] + ps[4][:30])  # a shared head
    got, core = run_engine(model, get_backend("hip"), None, ps, 25, **(KW | kw))
    exp, other = run_engine(model, PlainAttention(), None, ps, 25, **(KW | kw))
    assert core.stats().num_preemptions == other.stats().num_preemptions
    assert_greedy_match(got, exp)


@pytest.mark.parametrize("graphs", [False, (2, 8)])
@pytest.mark.parametrize("form", FORMS[:2], ids=["reference", "yarn"])
def test_forks_and_compactions(hip, graphs, form):
    # requests that fork on the way, the pool compacted every few steps or not: the same tokens.  A fork's tokens are its parent's
    # where it picks the best token as well
    from minillm.attention import get_backend
    from minillm.engine.core import AddRequest, EngineCore

    model = make_model(41, **form)
    model.set_backend(get_backend("hip"))
    runs = []
    for compacts in (False, True):
        rng = random.Random(5)
        core = EngineCore(model, decode_graphs=graphs, **(KW | dict(num_kv_blocks=80)))
        for i, (p, n) in enumerate(zip(prompts(5, 5, 150, seed=42), (40, 12, 33, 25, 60))):
            core.add_request(AddRequest(f"r{i}", p, n, ignore_eos=True))
        outs, forked, at, moved = {}, {}, 0, 0
        while core.has_work():
            for o in core.step().outputs:
                outs.setdefault(o.req_id, []).extend(o.new_token_ids)
            at += 1
            if at in (6, 11):
                name = sorted(r.req_id for r in core.scheduler.running)[0]
                core.fork(name, f"{name}+{at}")
                forked[f"{name}+{at}"] = (name, len(outs[name]))
            if compacts and rng.random() < 0.4:
                before = [list(r.block_ids) for r in core.scheduler.running]
                core.compact()
                moved += before != [r.block_ids for r in core.scheduler.running]
            core.check_blocks()
        assert not compacts or moved >= 2
        assert len(forked) == 2
        for child, (parent, since) in forked.items():
            assert outs[child] == outs[parent][since:]
        runs.append(outs)
    assert runs[0] == runs[1]


def test_pages_past_32_bits(hip):
    # a pool of more than 4 GiB of codes: append, attention, read back and copies at its far end, against the same rows at its front
    from minillm.attention import get_backend
    from minillm.attention.metadata import AttentionMetadata, SeqStep
    from test_gpu_fp8_blocks import make_cache

    blocks, hkv, h = 290000, 8, 32
    cache, be = make_cache(hkv, blocks), get_backend("hip")
    rows, need = [(100, 1), (700, 1), (33, 90), (0, 20)], [7, 44, 8, 2]
    g = torch.Generator().manual_seed(9)
    total, outs, values = sum(c + n for c, n in rows), [], []
    k, v = (torch.randn(total, hkv, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    q = torch.randn(sum(n for _, n in rows), h, 128, generator=g).bfloat16().to(DEV)
    for base in (0, blocks - sum(need)):
        ids = list(range(base, base + sum(need)))
        random.Random(1).shuffle(ids)
        tables = [[ids.pop() for _ in range(w)] for w in need]
        every = AttentionMetadata.build([SeqStep(0, c + n, t) for (c, n), t in zip(rows, tables)], 16, DEV)
        be.append(k, v, cache.k[0], cache.v[0], every, **cache.scales(0))
        meta = AttentionMetadata.build([SeqStep(c, n, t) for (c, n), t in zip(rows, tables)], 16, DEV)
        out = torch.empty_like(q)
        be.attend(q, cache.k[0], cache.v[0], meta, out, **cache.scales(0))
        outs.append(out)
        values.append(cache.read(0, every.slot_mapping))
    assert torch.equal(bits(outs[0]), bits(outs[1]))
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(*values))
    cache.copy_blocks([blocks - 1, blocks - 5], [blocks - 70, 100])
    for t in (cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0]):
        raw = t.view(torch.uint8)
        assert torch.equal(raw[blocks - 70], raw[blocks - 1]) and torch.equal(raw[100], raw[blocks - 5])
