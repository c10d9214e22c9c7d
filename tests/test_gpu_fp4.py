"""GPU parity of the 4-bit KV pool path (e2m1 codes, e8m0 block scales) against plain definitions in float64.

- append (`mllm_kv_append_fp4`, the 4-bit form of `mllm_qk_norm_rope_kv_append`) and read-back (`mllm_kv_read_fp4`): every
  quantised value identical to the definition's, over every 16-bit input pattern;
- attention (`mllm_paged_decode_fp4`, `mllm_merge_splits`, `mllm_paged_prefill_fp4`): against softmax(q k^T / sqrt(Dh)) v in
  float64 over the pool's values.

The attention's tolerance counts its roundings.  P is rounded to the 16-bit type, half a step each: sum_j p_j v_j is off by at
most eps / 2 of sum_j p_j |v_j|; the output by eps / 2 of itself.  Scores and sums are fp32: a score s is off by at most
(Dh + 4) 2^-24 of sum_d |q_d k_d| / sqrt(Dh), and the weights by that and 2^-21 (exp2 of an argument up to 2^8 and the
sums).  With A = sum_j p_j |v_j| the bound is eps/2 |out| + (eps/2 + 2 D + 2^-20) A, D the largest score error of the row.
"""

import math

import pytest
import torch

from harness import bits
from naive import causal_allowed

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
SCALE_RANGE = {torch.bfloat16: (1, 252), torch.float16: (104, 140)}


def quantised(x):
    """x [..., Dh] 16-bit on the CPU -> the float64 values a 4-bit pool holds for it, and the scale exponents."""
    lo, hi = SCALE_RANGE[x.dtype]
    b = x.double().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.floor(torch.log2(amax.clamp_min(2.0 ** -140) / 7)) + 1, -200.0)  # least 2^e > amax / 7
    e = e.nan_to_num(0.0, 0.0).clamp(lo - 127, hi - 127)
    y = (b / torch.exp2(e)).abs().nan_to_num(0.0, 6.0)
    # nearest of the grid, a tie to the even code
    d = (y[..., None] - GRID).abs()
    near = d == d.amin(-1, keepdim=True)
    odd_first = near.clone()
    odd_first[..., 1::2] &= ~near[..., 0::2].any(-1, keepdim=True)  # an odd code only where no even one is as near
    v = GRID[odd_first.double().argmax(-1)] * torch.exp2(e) * torch.where(torch.signbit(b), -1.0, 1.0)
    bad = ~torch.isfinite(b).all(-1, keepdim=True)
    v = torch.where(bad, math.nan, v)
    e = torch.where(bad, 128.0, e)[..., 0] + 127
    return v.flatten(-2), e.to(torch.uint8)


def make_cache(hkv, num_blocks, bs=16, layers=1, dh=128):
    from minillm.cache.paged import PagedKVCache
    from minillm.model.config import LlamaConfig

    cfg = LlamaConfig(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=layers,
                      num_attention_heads=hkv, num_key_value_heads=hkv, head_dim=dh, rms_norm_eps=1e-5, rope_theta=1e4)
    return PagedKVCache(cfg, num_blocks, DEV, FP4, block_size=bs)


class Slots:
    """What `append` reads of a step's metadata."""

    def __init__(self, slots):
        self.slot_mapping = slots


def append(cache, k, v, slots):
    from minillm.attention import get_backend

    get_backend("hip").append(k, v, cache.k[0], cache.v[0], Slots(slots), **cache.scales(0))


def same(got, want):
    """Equal values, NaN where NaN."""
    return torch.equal(got.double().cpu().nan_to_num(-12345.0), want.nan_to_num(-12345.0))


# ------------------------------------------------------------------ append and read


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_every_16bit_pattern(hip, dtype):
    # every pattern (subnormals, infinities and NaN included) in blocks of neighbours, so that each sets or nearly sets its
    # block's scale, and once more shuffled, so that blocks mix magnitudes
    pat = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    perm = torch.randperm(65536, generator=torch.Generator().manual_seed(0))
    k, v = pat.reshape(256, 2, 128), pat[perm].reshape(256, 2, 128)
    v = torch.where(torch.isfinite(v), v, torch.ones_like(v))
    slots = torch.randperm(512, generator=torch.Generator().manual_seed(1))[:256].to(DEV)
    cache = make_cache(2, 32)
    append(cache, k.to(DEV), v.to(DEV), slots)
    for got, x in zip(cache.read(0, slots, dtype), (k, v)):
        want, _ = quantised(x)
        assert same(got, want)
    # the scales themselves, at their places
    ks, vs = cache.k_scale[0].view(torch.uint8).cpu(), cache.v_scale[0].view(torch.uint8).cpu()
    for i in (0, 17, 255):
        s = int(slots[i])
        assert torch.equal(ks.view(512, 4, 2)[s], quantised(k[i])[1].t())
        assert torch.equal(vs[s // 16, :, :, s % 16], quantised(v[i])[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hkv,dh,bs,n", [(8, 128, 16, 1), (1, 64, 16, 37), (3, 192, 32, 50), (8, 128, 64, 333), (5, 128, 16, 7)])
def test_append_shapes_strides_and_slots(hip, dtype, hkv, dh, bs, n):
    # views into a joint projection, tokens without a slot, slots outside the pool; nothing else of the pool changes
    g = torch.Generator().manual_seed(n)
    blocks = -(-n // bs) + 2
    qkv = (torch.randn(n, 4 * hkv, dh, generator=g) * torch.logspace(-3, 3, 4 * hkv)[:, None]).to(dtype).to(DEV)
    k, v = qkv[:, hkv:2 * hkv], qkv[:, 3 * hkv:]
    slots = torch.randperm(blocks * bs, generator=g)[:n]
    if n > 4:
        slots[1], slots[n // 2] = -1, blocks * bs + 5
    slots = slots.to(DEV)
    cache = make_cache(hkv, blocks, bs, dh=dh)
    fill = torch.randint(0, 256, (blocks, bs, hkv, dh // 2), generator=g, dtype=torch.uint8).to(DEV)
    for p in (cache.k[0], cache.v[0]):
        p.view(torch.uint8).copy_(fill)
    append(cache, k, v, slots)
    got_k, got_v = cache.read(0, slots, dtype)
    inside = ((slots >= 0) & (slots < blocks * bs)).cpu()
    for got, x in ((got_k, k), (got_v, v)):
        want = torch.where(inside[:, None, None], quantised(x.cpu())[0], 0.0)  # a slot outside reads as zeros
        assert same(got, want)
    untouched = torch.ones(blocks * bs, dtype=torch.bool)
    untouched[slots.cpu()[inside]] = False
    for p in (cache.k[0], cache.v[0]):
        assert torch.equal(p.view(torch.uint8).flatten(0, 1).cpu()[untouched], fill.flatten(0, 1).cpu()[untouched])


# ------------------------------------------------------------------ attention


def step(rows, h, hkv, dtype, bs=16, seed=0, kv=None, junk=True, spare=1, scale_q=1.0):
    """A step of `rows` (cached, new) over a pool whose unowned slots hold junk (random codes, NaN scales included): the
    backend's output and the float64 one with its error bound."""
    from minillm.attention import get_backend
    from minillm.attention.metadata import AttentionMetadata, SeqStep

    g = torch.Generator().manual_seed(seed)
    need = [-(-(c + n) // bs) for c, n in rows]
    ids = torch.randperm(sum(need) + spare, generator=g).tolist()
    tables = [[ids.pop() for _ in range(w)] for w in need]
    cache = make_cache(hkv, sum(need) + spare, bs)
    if junk:
        for p, s in ((cache.k[0], cache.k_scale[0]), (cache.v[0], cache.v_scale[0])):
            p.view(torch.uint8).copy_(torch.randint(0, 256, p.shape, generator=g, dtype=torch.uint8))
            s.view(torch.uint8).copy_(torch.where(torch.rand(s.shape, generator=g) < 0.5, 255, 130).to(torch.uint8))
    meta = AttentionMetadata.build([SeqStep(c, n, t) for (c, n), t in zip(rows, tables)], bs, DEV)
    slots = torch.cat([torch.tensor([t[p // bs] * bs + p % bs for p in range(c + n)]) for (c, n), t in zip(rows, tables)])
    total = sum(c + n for c, n in rows)
    k, v = kv(total) if kv else (torch.randn(total, hkv, 128, generator=g) for _ in range(2))
    k, v = k.to(dtype).to(DEV), v.to(dtype).to(DEV)
    append(cache, k, v, slots.to(DEV))
    q = (torch.randn(sum(n for _, n in rows), h, 128, generator=g) * scale_q).to(dtype).to(DEV)
    out = torch.full_like(q, 7.0)
    backend = get_backend("hip")
    backend.attend(q, cache.k[0], cache.v[0], meta, out, **cache.scales(0))
    kd, vd = (t.double() for t in cache.read(0, slots.to(DEV), dtype))
    ref, bound = torch.empty(q.shape, dtype=torch.float64), torch.empty(q.shape, dtype=torch.float64)
    eps = torch.finfo(dtype).eps
    per, at, q0 = h // hkv, 0, 0
    for c, n in rows:
        allowed = causal_allowed(n, c + n).to(DEV)
        for x in range(hkv):
            kk, vv = kd[at:at + c + n, x].contiguous(), vd[at:at + c + n, x].contiguous()
            for y in range(per):
                qq = q[q0:q0 + n, x * per + y].double()
                s = (qq @ kk.t().contiguous()) / math.sqrt(128)
                p = torch.softmax(s.masked_fill(~allowed, -math.inf), -1)
                o, a = p @ vv, p @ vv.abs()
                ds = (132 * 2.0 ** -24 * (qq.abs() @ kk.abs().t().contiguous()) / math.sqrt(128)).masked_fill(~allowed, 0).amax(-1)
                ref[q0:q0 + n, x * per + y] = o.cpu()
                bound[q0:q0 + n, x * per + y] = (eps / 2 * o.abs() + (eps / 2 + 2 * ds[:, None] + 2.0 ** -20) * a).cpu()
        at, q0 = at + c + n, q0 + n
    return out.double().cpu(), ref, bound, (backend, cache, meta, q)


def check(out, ref, bound):
    worst = ((out - ref).abs() / bound.clamp_min(1e-30)).max().item()
    assert worst <= 1.0, f"error {worst:.3f} of its bound"


HEADS = [(32, 8), (16, 2), (8, 8), (16, 1), (4, 4), (12, 4), (10, 5), (3, 3), (14, 2)]


@pytest.mark.parametrize("h,hkv", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_heads(hip, h, hkv, dtype):
    # one token, a page less and more one, lengths over several bins
    check(*step([(0, 1), (14, 1), (15, 1), (16, 1), (200, 1), (777, 1)], h, hkv, dtype, seed=h)[:3])


@pytest.mark.parametrize("bs", [16, 32, 64])
def test_decode_block_sizes(hip, bs):
    check(*step([(0, 1), (31, 1), (500, 1), (63, 1), (1200, 1)], 32, 8, torch.bfloat16, bs=bs, seed=bs)[:3])


def test_decode_many_rows_and_a_long_one(hip):
    rows = [(int(x), 1) for x in torch.randint(0, 700, (150,), generator=torch.Generator().manual_seed(3))] + [(30000, 1)]
    check(*step(rows, 32, 8, torch.bfloat16, seed=4)[:3])


@pytest.mark.parametrize("h,hkv", [(32, 8), (8, 8), (16, 2), (16, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prefill_heads(hip, prefill_rows, h, hkv, dtype):
    check(*step([(0, 2), (0, 65), (17, 130), (300, 33), (1000, 16)], h, hkv, dtype, seed=h + 1)[:3])


@pytest.mark.parametrize("bs", [16, 32, 128])
def test_mixed_step_block_sizes(hip, prefill_rows, bs):
    check(*step([(100, 1), (0, 300), (129, 1), (640, 200), (0, 1)], 32, 8, torch.bfloat16, bs=bs, seed=bs + 7)[:3])


@pytest.mark.parametrize("rows", [[(300, 1)] * 3, [(40, 100)] * 2])
def test_loud_dims_and_sharp_softmax(hip, rows):
    # some dims of the keys 30 times the others and queries 4 times as long: weights close to one-hot, scores in the hundreds
    def kv(n):
        g = torch.Generator().manual_seed(9)
        k = torch.randn(n, 8, 128, generator=g)
        k[..., ::41] *= 30
        return k, torch.randn(n, 8, 128, generator=g) * torch.logspace(-2, 2, 128)

    check(*step(rows, 32, 8, torch.bfloat16, seed=11, kv=kv, scale_q=4.0)[:3])


def test_blocks_at_the_ends_of_the_range(hip):
    # fp16 values at the largest and among the smallest magnitudes stay finite and exact through attention
    def kv(n):
        g = torch.Generator().manual_seed(2)
        k = torch.randn(n, 2, 128, generator=g) * 2.0 ** -20
        v = torch.randn(n, 2, 128, generator=g).sign() * 65504.0
        v[1::2] = 2.0 ** -24
        return k, v

    for rows in ([(60, 1)], [(20, 30)]):
        out, ref, bound, _ = step(rows, 8, 2, torch.float16, seed=5, kv=kv)
        assert torch.isfinite(out).all()
        check(out, ref, bound)


def test_nan_and_inf_reach_only_their_own_head(hip):
    # an infinity in a key and a NaN in a value: the rows that see them are NaN in the query heads of that KV head only
    from minillm.attention import get_backend

    for rows in ([(50, 1), (20, 1)], [(10, 40), (20, 1)]):
        _, ref, bound, (backend, cache, meta, q) = step(rows, 32, 8, torch.bfloat16, seed=6)
        page = int(meta.block_tables[0, 0])
        cache.k_scale[0].view(torch.uint8)[page, 3, 2, 5] = 255
        cache.v_scale[0].view(torch.uint8)[page, 1, 0, 3] = 255
        out = torch.empty_like(q)
        backend.attend(q, cache.k[0], cache.v[0], meta, out, **cache.scales(0))
        n = rows[0][1]
        out = out.cpu()
        assert torch.isnan(out[:n, 20:24]).all()  # KV head 5
        assert torch.isnan(out[:n, 4:8, :32]).all() and torch.isfinite(out[:n, 4:8, 32:]).all()  # dim block 0 of head 1
        clean = [x for x in range(32) if not (20 <= x < 24 or 4 <= x < 8)]
        check(out[:n, clean].double(), ref[:n, clean], bound[:n, clean])
        check(out[n:].double(), ref[n:], bound[n:])


def test_output_rows_of_other_sequences_stay(hip):
    # rows behind the last sequence and a strided output: only the step's own elements are written
    _, ref, bound, (backend, cache, meta, q) = step([(77, 1), (3, 20)], 32, 8, torch.bfloat16, seed=8)
    wide = torch.full((q.shape[0] + 5, 40, 128), 3.0, dtype=q.dtype, device=DEV)
    backend.attend(q, cache.k[0], cache.v[0], meta, wide[:q.shape[0], 4:36], **cache.scales(0))
    check(wide[:q.shape[0], 4:36].double().cpu(), ref, bound)
    wide[:q.shape[0], 4:36] = 3.0
    assert bool((wide == 3.0).all())


def test_attend_in_one_call_and_launch_by_launch(hip):
    # a contiguous output goes in one host call, a strided one and a mixed step on two streams launch by launch
    *_, (backend, cache, meta, q) = step([(300, 1), (50, 20), (2000, 1), (0, 7)], 32, 8, torch.bfloat16, seed=9)
    out, wide = torch.empty_like(q), torch.empty(q.shape[0], 40, 128, dtype=q.dtype, device=DEV)
    two = torch.empty_like(q)
    backend.attend(q, cache.k[0], cache.v[0], meta, out, **cache.scales(0))
    backend.attend(q, cache.k[0], cache.v[0], meta, wide[:, 4:36], **cache.scales(0))
    backend.overlap_mixed = True
    backend.attend(q, cache.k[0], cache.v[0], meta, two, **cache.scales(0))
    assert torch.equal(bits(out), bits(wide[:, 4:36].contiguous())) and torch.equal(bits(out), bits(two))


def test_forward_equals_append_and_attend(hip):
    # the layer's one host call, without and with the rotation: the pool's bytes and the output of the separate calls
    from minillm.model.llama import apply_rotary

    g = torch.Generator().manual_seed(21)
    for dtype in (torch.bfloat16, torch.float16):
        *_, (backend, cache, meta, q) = step([(100, 1), (30, 40), (0, 1)], 32, 8, dtype, seed=20)
        n = q.shape[0]
        k, v = (torch.randn(n, 8, 128, generator=g).to(dtype).to(DEV) for _ in range(2))
        ang = torch.randn(n, 64, generator=g).repeat(1, 2)
        cos, sin = ang.cos().to(dtype).to(DEV), ang.sin().to(dtype).to(DEV)
        pools = (cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0])
        start = [p.view(torch.uint8).clone() for p in pools]

        def fresh():
            for p, s in zip(pools, start):
                p.view(torch.uint8).copy_(s)

        def state():
            return [p.view(torch.uint8).clone() for p in pools]

        fresh()
        backend.append(k, v, *pools[:2], meta, **cache.scales(0))
        want = torch.empty_like(q)
        backend.attend(q, *pools[:2], meta, want, **cache.scales(0))
        after = state()
        fresh()
        got = backend.forward(q, k, v, *pools[:2], meta, **cache.scales(0))
        assert torch.equal(bits(got), bits(want)) and all(torch.equal(a, b) for a, b in zip(state(), after))

        rot = [apply_rotary(x.transpose(0, 1)[None], cos[None], sin[None])[0].transpose(0, 1) for x in (q, k)]
        fresh()
        want = backend.forward(rot[0], rot[1], v, *pools[:2], meta, **cache.scales(0))
        after = state()
        fresh()
        got = backend.forward_rotary(q, k, v, cos, sin, *pools[:2], meta, **cache.scales(0))
        assert torch.equal(bits(got), bits(want)) and all(torch.equal(a, b) for a, b in zip(state(), after))
        fresh()
        q_rot = backend.rope_append(q, k, v, cos, sin, *pools[:2], meta, **cache.scales(0))
        assert torch.equal(bits(q_rot), bits(rot[0].contiguous())) and all(torch.equal(a, b) for a, b in zip(state(), after))


# partials that hold a NaN in each of their tiles, of how many: the first four of a head's eight; one that is alone in its
# group of the merge; every one of a group; the last; all
NAN_PARTIALS = [(6, (0, 1, 2, 3)), (8, (0, 1, 2, 3)), (9, (3,)), (12, (5,)), (15, (7,)), (20, (2, 10, 18)), (21, (20,)), (3, (0, 1, 2))]


@pytest.mark.parametrize("parts,bad", NAN_PARTIALS)
@pytest.mark.parametrize("others", [0, 100], ids=["alone", "among100"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_segments_of_nan_keys_reach_the_merged_row(hip, monkeypatch, parts, bad, others, dtype):
    # bins of two pages; with 100 other cut rows a workgroup of the merge serves eight heads
    monkeypatch.setenv("MLLM_PAGES_PER_SPLIT", "2")
    rows = [(32 * parts - 5, 1)] + [(60, 1)] * others
    _, ref, bound, (backend, cache, meta, q) = step(rows, 32, 8, dtype, seed=parts)
    merges = backend.plan(meta, 32, 8, 128, q.device, pool=2).merge_work.view(-1, 4).cpu()
    assert merges[merges[:, 0] == 0][:, 2].tolist() == [parts] and int((merges[:, 0] >= 0).sum()) == 1 + others
    pages = meta.block_tables[0].cpu().tolist()
    scales = cache.k_scale[0].view(torch.uint8)
    for p in bad:
        scales[pages[2 * p], 3, 2, 5] = 255
        scales[pages[2 * p + 1], 1, 0, 5] = 255
    out = torch.empty_like(q)
    backend.attend(q, cache.k[0], cache.v[0], meta, out, **cache.scales(0))
    out = out.cpu()
    assert torch.isnan(out[0, 20:24]).all()  # KV head 5
    clean = [x for x in range(32) if not 20 <= x < 24]
    check(out[:1, clean].double(), ref[:1, clean], bound[:1, clean])
    if others:
        check(out[1:].double(), ref[1:], bound[1:])


def test_layers_of_other_head_counts_share_a_steps_metadata(hip):
    # each call of one backend is what a backend of its own gives
    from minillm.attention.hip_backend import HipBackend

    *_, (backend, first, meta, q0) = step([(300, 1), (40, 9), (2000, 1)], 32, 8, torch.bfloat16, seed=13)
    g = torch.Generator().manual_seed(14)
    for h, hkv in ((8, 8), (8, 2), (32, 8), (32, 2), (4, 4)):
        cache = make_cache(hkv, first.num_blocks)
        n = first.num_blocks * 16
        k, v = (torch.randn(n, hkv, 128, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
        append(cache, k, v, torch.arange(n, device=DEV))
        q = torch.randn(q0.shape[0], h, 128, generator=g).to(torch.bfloat16).to(DEV)
        rows = torch.full((q0.shape[0] + 1, h, 128), 3.0, dtype=q.dtype, device=DEV)  # the last row lies behind the step
        want = torch.empty_like(q)
        backend.attend(q, cache.k[0], cache.v[0], meta, rows[:-1], **cache.scales(0))
        HipBackend().attend(q, cache.k[0], cache.v[0], meta, want, **cache.scales(0))
        assert torch.equal(bits(rows[:-1]), bits(want)) and bool((rows[-1] == 3.0).all())
