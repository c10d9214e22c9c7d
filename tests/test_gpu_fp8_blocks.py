"""GPU parity of the 8-bit KV pool with a scale for each page and head against plain definitions in float64.

- append (`mllm_kv_append_fp8_blocks`, its form of `mllm_qk_norm_rope_kv_append`) and read-back (`mllm_kv_read_fp8_blocks`):
  codes and scales identical to the definition's, however the tokens of a page come in;
- attention (`mllm_paged_decode_fp8_blocks`, `mllm_paged_prefill_fp8_blocks`): against softmax(q k^T / sqrt(Dh)) v in float64
  over the pool's values.

The attention's tolerance counts its roundings.  P is rounded to the 16-bit type, half a step each: sum_j p_j v_j is off by at
most eps / 2 of sum_j p_j |v_j|; the output by eps / 2 of itself.  Scores and sums are fp32: a score s is off by at most
(Dh + 4) 2^-24 of sum_d |q_d k_d| / sqrt(Dh), and the weights by that and 2^-21 (exp2 of an argument up to 2^8 and the
sums).  With A = sum_j p_j |v_j| the bound is eps/2 |out| + (eps/2 + 2 D + 2^-20) A, D the largest score error of the row.
In rows of one new token P is the sum of two 16-bit values, the second the first one's rounding error (exact in fp32) rounded
again: (eps/2)^2 A there.
In fp16 a P below 2^-14 is subnormal, where half a step is 2^-25 whatever p is.  P is taken relative to a maximum that some key
of the row has reached, so its sum, by which the output is divided, is at least 1: 2^-25 sum_j |v_j| more.
"""

import math
import random

import pytest
import torch

from harness import bits
from naive import causal_allowed

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP8, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
SCALE_RANGE = {torch.bfloat16: (10, 246), torch.float16: (112, 134)}
DTYPES = [torch.bfloat16, torch.float16]


def to_e4m3(x):
    """x (float64) to the nearest e4m3 value, ties to the even multiple, at most 448; not finite: NaN."""
    a = x.abs().nan_to_num(0.0, 0.0)
    e = torch.floor(torch.log2(a.clamp_min(2.0 ** -300))).clamp_min(-6.0)
    e = torch.where(torch.exp2(e) > a, e - 1, torch.where(torch.exp2(e + 1) <= a, e + 1, e)).clamp_min(-6.0)
    step = torch.exp2(e - 3)
    y = (torch.round(a / step) * step).clamp_max(448.0)  # torch.round: ties to even
    return torch.where(torch.isfinite(x), torch.where(torch.signbit(x), -y, y), math.nan)


def exponent(x, dtype):
    """The scale exponent of tokens x [n, Hkv, Dh]: [Hkv] (biased)."""
    lo, hi = SCALE_RANGE[dtype]
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).double().amax(dim=(0, 2))
    return torch.tensor([next((e for e in range(lo, hi) if v <= math.ldexp(448.0, e - 127)), hi) for v in a.tolist()])


class PoolByDefinition:
    """One pool (K or V) as the definition says: values of the codes and exponents."""

    def __init__(self, blocks, bs, hkv, dtype):
        self.codes = torch.zeros(blocks, bs, hkv, 128, dtype=torch.float64)
        self.e = torch.zeros(blocks, hkv, dtype=torch.int64)
        self.bs, self.dtype = bs, dtype

    def append(self, x, slots):
        x, i = x.cpu(), 0
        blocks = self.codes.shape[0]
        slots = slots.tolist()
        while i < len(slots):
            n = 1
            if not 0 <= slots[i] < blocks * self.bs:
                i += 1
                continue
            page, at = divmod(slots[i], self.bs)
            while i + n < len(slots) and at + n < self.bs and slots[i + n] == slots[i] + n:
                n += 1
            rows = x[i:i + n]
            e = exponent(rows, self.dtype)
            if at:
                e = torch.maximum(e, self.e[page])
                down = torch.exp2((self.e[page] - e).double())[:, None]
                self.codes[page, :at] = torch.where(down < 1, to_e4m3(self.codes[page, :at] * down), self.codes[page, :at])
            self.e[page] = e
            self.codes[page, at:at + n] = to_e4m3(rows.double() / torch.exp2((e - 127).double())[:, None])
            i += n

    def values(self, slots):
        page, at = slots // self.bs, slots % self.bs
        return self.codes[page, at] * torch.exp2((self.e[page] - 127).double())[..., None]


def make_cache(hkv, num_blocks, bs=16, layers=1):
    from minillm.cache.paged import PagedKVCache
    from minillm.model.config import LlamaConfig

    cfg = LlamaConfig(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=layers,
                      num_attention_heads=hkv, num_key_value_heads=hkv, head_dim=128, rms_norm_eps=1e-5, rope_theta=1e4)
    return PagedKVCache(cfg, num_blocks, DEV, FP8, block_size=bs, block_scales=True)


class Slots:
    """What `append` reads of a step's metadata."""

    def __init__(self, slots):
        self.slot_mapping = slots


def append(cache, k, v, slots):
    from minillm.attention import get_backend

    get_backend("hip").append(k, v, cache.k[0], cache.v[0], Slots(slots.to(DEV)), **cache.scales(0))


def same(got, want):
    """Equal values, NaN where NaN."""
    return torch.equal(got.double().cpu().nan_to_num(-12345.0), want.nan_to_num(-12345.0))


def assert_pool(cache, of_k, of_v, slots):
    """Codes of `slots` and every scale of the pages they lie in, bit for bit."""
    pages = (slots // of_k.bs).unique()
    for codes, scale, want in ((cache.k[0], cache.k_scale[0], of_k), (cache.v[0], cache.v_scale[0], of_v)):
        assert torch.equal(scale.view(torch.uint8).cpu().long()[pages], want.e[pages])
        got = codes.view(torch.uint8).flatten(0, 1).cpu()[slots].view(FP8)
        assert same(got, want.codes.flatten(0, 1)[slots])


# ------------------------------------------------------------------ append and read


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_every_16bit_pattern(hip, dtype):
    # every pattern (subnormals, infinities and NaN included): each page holds neighbours, which set or nearly set its scale;
    # V the same shuffled, so that pages mix magnitudes
    pat = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    perm = torch.randperm(65536, generator=torch.Generator().manual_seed(0))
    k, v = pat.reshape(256, 2, 128), pat[perm].reshape(256, 2, 128)
    small = torch.isfinite(v) & (v.double().abs() < 2.0 ** 6)
    v = torch.where(small, v, torch.ones_like(v))
    pages = torch.randperm(16, generator=torch.Generator().manual_seed(1))
    slots = (pages[:, None] * 16 + torch.arange(16)).flatten()
    cache = make_cache(2, 16)
    append(cache, k.to(DEV), v.to(DEV), slots)
    of_k, of_v = PoolByDefinition(16, 16, 2, dtype), PoolByDefinition(16, 16, 2, dtype)
    of_k.append(k, slots), of_v.append(v, slots)
    assert_pool(cache, of_k, of_v, slots)
    for got, want in zip(cache.read(0, slots.to(DEV), dtype), (of_k, of_v)):
        assert same(got, want.values(slots))


def random_rows(n, hkv, g, dtype, spread=3.0):
    """Rows whose loudness differs by token and head, a few infinities and NaN among them."""
    x = torch.randn(n, hkv, 128, generator=g) * torch.exp2(spread * torch.randn(n, hkv, 1, generator=g))
    x = torch.where(torch.rand(x.shape, generator=g) < 1e-4, torch.tensor(math.inf), x)
    return torch.where(torch.rand(x.shape, generator=g) < 1e-4, torch.tensor(math.nan), x).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,bs,most,seed", [(8, 16, 1, 1), (3, 16, 5, 2), (1, 32, 40, 3), (2, 64, 100, 4), (8, 16, 700, 5),
                                              (2, 16, 3000, 6)])
def test_append_in_steps(hip, dtype, hkv, bs, most, seed):
    # sequences that grow by up to `most` tokens a step, several to a step, until pages have come in in many ways; then their
    # pages serve others.  Codes, scales and values after every step
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    blocks = 4 * (-(-4 * most // bs)) + 24
    cache = make_cache(hkv, blocks, bs)
    of_k, of_v = PoolByDefinition(blocks, bs, hkv, dtype), PoolByDefinition(blocks, bs, hkv, dtype)
    seqs = []  # [table, tokens so far]
    free = list(range(blocks))
    rng.shuffle(free)
    for step in range(12):
        if len(seqs) < 4:
            seqs.append([[], 0])
        elif step == 7:  # a sequence ends
            free += seqs.pop(1)[0]
        slots = []
        for seq in seqs:
            for _ in range(rng.randint(1, most)):
                if seq[1] % bs == 0 and seq[1] // bs == len(seq[0]):
                    if len(free) < 2:
                        break
                    seq[0].append(free.pop())
                slots.append(seq[0][seq[1] // bs] * bs + seq[1] % bs)
                seq[1] += 1
        if not slots:
            continue
        slots = torch.tensor(slots)
        qkv = torch.cat([random_rows(len(slots), hkv, g, dtype) for _ in range(3)], dim=1).to(DEV)
        k, v = qkv[:, :hkv], qkv[:, 2 * hkv:]  # views into a joint projection
        append(cache, k, v, slots)
        of_k.append(k, slots), of_v.append(v, slots)
        held = torch.tensor([t[p // bs] * bs + p % bs for t, n in seqs for p in range(n)])
        assert_pool(cache, of_k, of_v, held)
    for got, want in zip(cache.read(0, held.to(DEV), dtype), (of_k, of_v)):
        assert same(got, want.values(held))


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_leaves_the_rest(hip, dtype):
    # tokens without a slot and slots outside the pool; pages and slots that no token has keep their bytes
    g = torch.Generator().manual_seed(3)
    cache = make_cache(4, 6)
    for p, s in ((cache.k[0], cache.k_scale[0]), (cache.v[0], cache.v_scale[0])):
        p.view(torch.uint8).copy_(torch.randint(0, 256, p.shape, generator=g, dtype=torch.uint8))
        s.view(torch.uint8).copy_(torch.randint(0, 256, s.shape, generator=g, dtype=torch.uint8))
    before = [x.view(torch.uint8).cpu().clone() for x in (cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0])]
    slots = torch.tensor([-1, 16, 17, 18, -1, 96, 97, 48 + 16, 5000000000, -7, 32, 33])
    rows = [random_rows(len(slots), 4, g, dtype).to(DEV) for _ in range(2)]
    append(cache, *rows, slots)
    inside = (slots >= 0) & (slots < 96)
    kept, pages = torch.ones(96, dtype=torch.bool), torch.ones(6, dtype=torch.bool)
    kept[slots[inside]], pages[(slots[inside] // 16)] = False, False
    after = [x.view(torch.uint8).cpu() for x in (cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0])]
    for a, b in zip(after[:2], before[:2]):
        assert torch.equal(a.flatten(0, 1)[kept], b.flatten(0, 1)[kept])
    for a, b in zip(after[2:], before[2:]):
        assert torch.equal(a[pages], b[pages])
    of_k = PoolByDefinition(6, 16, 4, dtype)
    of_k.append(rows[0], slots)
    got = cache.read(0, slots.to(DEV), dtype)[0].double().cpu()
    assert same(got[inside], of_k.values(slots[inside]))
    assert (got[~inside] == 0).all()
    empty = torch.empty(0, dtype=torch.int64)
    append(cache, rows[0][:0], rows[1][:0], empty)  # nothing to append, nothing to read
    assert cache.read(0, empty.to(DEV))[0].shape == (0, 4, 128)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,start", [(1, 0), (7, 9), (200, 3), (1500, 21)])
def test_rope_append_equals_rotary_then_append(hip, dtype, n, start):
    from minillm.attention import get_backend
    from minillm.model.llama import apply_rotary

    h, hkv, g = 8, 2, torch.Generator().manual_seed(n)
    blocks = -(-(start + n) // 16)
    qkv = torch.randn(n, h + 2 * hkv, 128, generator=g).to(dtype).to(DEV)
    q, k, v = qkv.split((h, hkv, hkv), dim=1)
    ang = torch.randn(n, 64, generator=g) * 3
    cos, sin = (torch.cat([f(ang)] * 2, dim=1).to(dtype).to(DEV) for f in (torch.cos, torch.sin))
    slots = torch.arange(start, start + n).to(DEV)
    first = [torch.randn(start, hkv, 128, generator=g).to(dtype).to(DEV) for _ in range(2)]
    caches = [make_cache(hkv, blocks) for _ in range(2)]
    for c in caches:
        if start:
            append(c, *first, torch.arange(start))

    class Meta(Slots):
        block_size, query_start_loc = 16, [0, n]

    be = get_backend("hip")
    rot = [apply_rotary(x.transpose(0, 1)[None], cos[None], sin[None])[0].transpose(0, 1) for x in (q, k)]
    append(caches[1], rot[1], v, slots)
    got = be.rope_append(q, k, v, cos, sin, caches[0].k[0], caches[0].v[0], Meta(slots), **caches[0].scales(0))
    assert torch.equal(bits(got), bits(rot[0].contiguous()))
    for a, b in zip((caches[0].k[0], caches[0].v[0], caches[0].k_scale[0], caches[0].v_scale[0]),
                    (caches[1].k[0], caches[1].v[0], caches[1].k_scale[0], caches[1].v_scale[0])):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 33, 1100])
def test_norm_rope_append(hip, dtype, n):
    # q and the pool's keys against the formula in float64: q rounds once (half a step), a key once more to e4m3 (2^-4 of it, or
    # half a step of the subnormal grid, 2^-10 of the scale); the fp32 arithmetic before takes 2^-20
    from minillm.attention import get_backend

    h, hkv, eps, g = 8, 4, 1e-5, torch.Generator().manual_seed(n)
    cache = make_cache(hkv, -(-n // 16))
    qkv = (torch.randn(n, h + 2 * hkv, 128, generator=g) * torch.logspace(-2, 2, h + 2 * hkv)[:, None]).to(dtype).to(DEV)
    q, k, v = qkv.split((h, hkv, hkv), dim=1)
    wq, wk = ((1 + 0.2 * torch.randn(128, generator=g)).to(dtype).to(DEV) for _ in range(2))
    ang = torch.randn(n, 64, generator=g) * 3
    cos, sin = (torch.cat([f(ang)] * 2, dim=1).to(dtype).to(DEV) for f in (torch.cos, torch.sin))

    class Meta(Slots):
        block_size, query_start_loc = 16, [0, n]

    got = get_backend("hip").rope_append(q, k, v, cos, sin, cache.k[0], cache.v[0], Meta(torch.arange(n).to(DEV)),
                                         qk_norm=(wq, wk, eps), **cache.scales(0))

    def formula(x, w):
        y = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps) * w.double()
        turn = torch.cat([-y[..., 64:], y[..., :64]], dim=-1)
        c, s = cos.double()[:, None], sin.double()[:, None]
        return y * c + turn * s, (y * c).abs() + (turn * s).abs()

    half = torch.finfo(dtype).eps / 2
    ref, size = formula(q, wq)
    assert ((got.double() - ref).abs() <= half * ref.abs() + 2.0 ** -20 * size + 2.0 ** -25).all()
    ref, size = formula(k, wk)
    gk, gv = cache.read(0, torch.arange(n).to(DEV), dtype)
    unit = torch.exp2(cache.k_scale[0].view(torch.uint8).double() - 127)[torch.arange(n).to(DEV) // 16][..., None]
    off = half * ref.abs() + 2.0 ** -20 * size + 2.0 ** -25
    assert ((gk.double() - ref).abs() <= off + 2.0 ** -4 * (ref.abs() + off) + 2.0 ** -10 * unit).all()
    of_v = PoolByDefinition(-(-n // 16), 16, hkv, dtype)
    of_v.append(v, torch.arange(n))
    assert same(gv, of_v.values(torch.arange(n)))


# ------------------------------------------------------------------ attention


def step(rows, h, hkv, dtype, bs=16, seed=0, kv=None, spare=1, scale_q=1.0):
    """A step of `rows` (cached, new) over a pool whose unowned slots hold junk (codes of NaN and scales of NaN included): the
    backend's output and the float64 one with its error bound."""
    from minillm.attention import get_backend
    from minillm.attention.metadata import AttentionMetadata, SeqStep

    g = torch.Generator().manual_seed(seed)
    need = [-(-(c + n) // bs) for c, n in rows]
    ids = torch.randperm(sum(need) + spare, generator=g).tolist()
    tables = [[ids.pop() for _ in range(w)] for w in need]
    cache = make_cache(hkv, sum(need) + spare, bs)
    for p, s in ((cache.k[0], cache.k_scale[0]), (cache.v[0], cache.v_scale[0])):
        p.view(torch.uint8).copy_(torch.randint(0, 256, p.shape, generator=g, dtype=torch.uint8))
        s.view(torch.uint8).fill_(255)
    meta = AttentionMetadata.build([SeqStep(c, n, t) for (c, n), t in zip(rows, tables)], bs, DEV)
    slots = torch.cat([torch.tensor([t[p // bs] * bs + p % bs for p in range(c + n)]) for (c, n), t in zip(rows, tables)])
    total = sum(c + n for c, n in rows)
    loud = torch.exp2(4 * torch.randn(2, total, hkv, 1, generator=g) - 3)
    k, v = kv(total) if kv else torch.randn(2, total, hkv, 128, generator=g).unbind()
    v = v * loud[1]
    k, v = k.to(dtype).to(DEV), v.to(dtype).to(DEV)
    append(cache, k, v, slots)
    q = (torch.randn(sum(n for _, n in rows), h, 128, generator=g) * scale_q).to(dtype).to(DEV)
    out = torch.full_like(q, 7.0)
    backend = get_backend("hip")
    backend.attend(q, cache.k[0], cache.v[0], meta, out, **cache.scales(0))
    kd, vd = (t.double() for t in cache.read(0, slots.to(DEV), dtype))
    ref, bound = torch.empty(q.shape, dtype=torch.float64), torch.empty(q.shape, dtype=torch.float64)
    eps = torch.finfo(dtype).eps
    tiny = torch.finfo(dtype).smallest_normal * eps  # half a step of a subnormal output is at most this
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
                low = 2.0 ** -25 * (allowed.double() @ vv.abs()) if dtype == torch.float16 else 0.0
                of_p = eps / 2 if n > 1 else (eps / 2) ** 2
                bound[q0:q0 + n, x * per + y] = (eps / 2 * o.abs() + (of_p + 2 * ds[:, None] + 2.0 ** -20) * a + tiny + low).cpu()
        at, q0 = at + c + n, q0 + n
    return out.double().cpu(), ref, bound, (backend, cache, meta, q)


def check(out, ref, bound):
    """NaN where the reference is (a value past fp16's range came in as an infinity), else within the bound."""
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(out), nan)
    worst = ((out - ref).abs() / bound)[~nan].max().item()
    assert worst <= 1.0, f"error {worst:.3f} of its bound"


HEADS = [(32, 8), (16, 2), (8, 8), (16, 1), (4, 4), (12, 4), (10, 5), (3, 3), (14, 2)]


@pytest.mark.parametrize("h,hkv", HEADS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_heads(hip, h, hkv, dtype):
    # one token, a page less and more one, lengths over several bins
    check(*step([(0, 1), (14, 1), (15, 1), (16, 1), (200, 1), (777, 1)], h, hkv, dtype, seed=h)[:3])


@pytest.mark.parametrize("bs", [16, 32, 64])
def test_decode_block_sizes(hip, bs):
    check(*step([(0, 1), (31, 1), (500, 1), (63, 1), (1200, 1)], 32, 8, torch.bfloat16, bs=bs, seed=bs)[:3])


def test_decode_many_rows_and_a_long_one(hip):
    rows = [(int(x), 1) for x in torch.randint(0, 700, (150,), generator=torch.Generator().manual_seed(3))] + [(30000, 1)]
    check(*step(rows, 32, 8, torch.bfloat16, seed=4)[:3])


@pytest.mark.parametrize("h,hkv", [(32, 8), (16, 1), (8, 8), (12, 3), (64, 2)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_and_mixed(hip, h, hkv, dtype, prefill_rows):
    # chunks that start within a page, end within a 64-key tile, of two tokens, without cached ones; decode rows beside them
    rows = [(0, 2), (5, 37), (63, 65), (0, 200), (130, 129), (300, 64)]
    if h // hkv <= 16:
        rows += [(40, 1), (900, 1)]
    check(*step(rows, h, hkv, dtype, seed=h + hkv)[:3])


@pytest.mark.parametrize("bs", [32, 64])
def test_prefill_block_sizes(hip, bs, prefill_rows):
    check(*step([(0, 100), (77, 33), (31, 64), (250, 300)], 32, 8, torch.bfloat16, bs=bs, seed=bs)[:3])


@pytest.mark.parametrize("h,hkv,bs", [(8, 2, 16), (6, 3, 16), (8, 1, 64), (10, 5, 32)])
def test_prefill_behind_long_contexts(hip, h, hkv, bs, prefill_rows):
    # ids and scales are taken 64 tiles (4,096 tokens) at a time: contexts that end around and behind such windows
    rows = [(3839, 2), (3900, 130), (4090, 300), (8100, 64), (9000, 40), (12345, 70)]
    check(*step(rows, h, hkv, torch.bfloat16, bs=bs, seed=hkv)[:3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_sharp_softmax(hip, dtype):
    # scores over hundreds: rows that one key wins, and the running maximum moves
    check(*step([(300, 1), (1000, 1), (17, 40), (0, 130)], 8, 2, dtype, seed=9, scale_q=30.0)[:3])


def test_scales_far_apart(hip):
    # pages of one row whose scales lie 2^200 apart: no scale of another page takes part
    def kv(total):
        g = torch.Generator().manual_seed(1)
        k, v = torch.randn(2, total, 2, 128, generator=g).unbind()
        page = (torch.arange(total) // 16 % 2)[:, None, None]
        return torch.where(page == 0, k, k * 2.0 ** -100), torch.where(page == 0, v * 2.0 ** 50, v * 2.0 ** -60)

    check(*step([(100, 1), (40, 20)], 8, 2, torch.bfloat16, seed=5, kv=kv)[:3])


def test_nan_key_reaches_its_own_rows_only(hip):
    # a NaN among a row's keys: that row's heads over that KV head, and no other
    from minillm.attention import get_backend

    _, _, _, (be, cache, meta, q) = step([(100, 1), (400, 1), (9, 1)], 8, 2, torch.bfloat16, seed=6)
    want = torch.empty_like(q)
    be.attend(q, cache.k[0], cache.v[0], meta, want, **cache.scales(0))
    slot = int(meta.kv_indices[int(meta.kv_indptr[1])]) * 16 + 3
    cache.k[0].view(torch.uint8).flatten(0, 1)[slot, 1, 7] = 0x7f
    out = torch.empty_like(q)
    get_backend("hip").attend(q, cache.k[0], cache.v[0], meta, out, **cache.scales(0))
    hit = torch.zeros(3, 8, dtype=torch.bool)
    hit[1, 4:] = True
    assert torch.isnan(out[hit.to(DEV)]).all() and torch.equal(out[~hit.to(DEV)], want[~hit.to(DEV)])


def test_other_stream_strided_q_and_out(hip):
    # attention on a side stream, of q inside a joint projection, into rows of a wider tensor (two launches instead of one call)
    out, ref, bound, (be, cache, meta, q) = step([(50, 1), (300, 1), (20, 30)], 8, 2, torch.bfloat16, seed=7)
    wide_q = torch.zeros(q.shape[0], 3, 8, 128, dtype=q.dtype, device=DEV)
    wide_q[:, 1] = q
    wide_out = torch.full((q.shape[0], 2, 8, 128), 3.0, dtype=q.dtype, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        be.attend(wide_q[:, 1], cache.k[0], cache.v[0], meta, wide_out[:, 1], **cache.scales(0))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(wide_out[:, 1].double().cpu(), out) and (wide_out[:, 0] == 3.0).all()


def test_captured_calls(hip):
    # append and attention in a graph, replayed with the program's own work between: every replay the eager call's bits
    _, _, _, (be, cache, meta, q) = step([(50, 1), (300, 1), (20, 30)], 8, 2, torch.bfloat16, seed=8)
    n = q.shape[0]
    rows = torch.randn(2, n, 2, 128, device=DEV).to(q.dtype)
    out = torch.empty_like(q)

    def body():
        be.append(rows[0], rows[1], cache.k[0], cache.v[0], meta, **cache.scales(0))
        be.attend(q, cache.k[0], cache.v[0], meta, out, **cache.scales(0))

    held = [x.view(torch.uint8).clone() for x in (cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    for seed in range(4):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rows.copy_(torch.randn(rows.shape, generator=g, device=DEV) * (1 + 3 * seed))
        q.copy_(torch.randn(q.shape, generator=g, device=DEV))
        got = []
        for run in (body, graph.replay):
            for x, was in zip((cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0]), held):
                x.view(torch.uint8).copy_(was)
            run()
            torch.cuda.synchronize()
            got.append([x.view(torch.uint8).clone() for x in (out, cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0])])
        assert all(torch.equal(a, b) for a, b in zip(*got))
