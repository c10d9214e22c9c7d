"""Appends of many tokens into 8-bit pools with block scales whose pages are of 32 and 64 tokens, against the definition: runs longer
than the 16 tokens that stay in registers, that begin anywhere in a page and in a window, beside short ones and tokens without a
slot; plain, rotated, and normed and rotated."""

import random

import pytest
import torch

from harness import bits
from test_gpu_fp8_blocks import DEV, DTYPES, PoolByDefinition, Slots, append, assert_pool, make_cache, random_rows, same
from test_gpu_fp8_blocks import test_append_in_steps as append_in_steps

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,bs,most,seed", [(2, 32, 1500, 7), (3, 64, 1500, 8), (1, 64, 4000, 9)])
def test_growing_sequences(hip, dtype, hkv, bs, most, seed):
    append_in_steps(hip, dtype, hkv, bs, most, seed)


def runs(rng, blocks, bs, at_least, longest):
    """Slots of a step of at least so many tokens: every page's tokens in one run, tokens without a slot between some."""
    pages, slots = list(range(blocks)), []
    rng.shuffle(pages)
    while len(slots) < at_least:
        page = pages.pop()
        first = rng.choice([0, 0, rng.randrange(bs)])
        n = min(bs - first, rng.choice([1, 2, 4, 5, 15, 16, 17, 31, 33, 48, 49, 63, 64, rng.randint(1, bs)]), longest)
        slots += range(page * bs + first, page * bs + first + n)
        if first + n == bs and page + 1 in pages and rng.random() < 0.5:  # the slots go on into the next page, a run of its own
            pages.remove(page + 1)
            slots += range((page + 1) * bs, (page + 1) * bs + rng.randint(1, bs))
        if rng.random() < 0.1:
            slots += [-1] * rng.randint(1, 5)
    return torch.tensor(slots)


def filled(rng, g, hkv, blocks, bs, dtype):
    """A cache whose pages hold tokens already, and what the definition says of it."""
    cache = make_cache(hkv, blocks, bs)
    of_k, of_v = (PoolByDefinition(blocks, bs, hkv, dtype) for _ in range(2))
    slots = torch.arange(blocks * bs)
    k, v = (random_rows(len(slots), hkv, g, dtype, spread=4.0) for _ in range(2))
    append(cache, k.to(DEV), v.to(DEV), slots)
    of_k.append(k, slots), of_v.append(v, slots)
    return cache, of_k, of_v


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,bs,longest,seed", [(1, 64, 64, 1), (3, 64, 64, 2), (2, 32, 32, 3), (2, 64, 20, 4), (8, 16, 16, 5), (1, 64, 64, 6)])
def test_runs_of_any_length(hip, dtype, hkv, bs, longest, seed):
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    blocks = 260 * 16 // bs + 30
    cache, of_k, of_v = filled(rng, g, hkv, blocks, bs, dtype)
    for step in range(3):
        slots = runs(rng, blocks, bs, 1025 + 17 * step, longest)
        k, v = (random_rows(len(slots), hkv, g, dtype, spread=4.0) for _ in range(2))
        append(cache, k.to(DEV), v.to(DEV), slots)
        of_k.append(k, slots), of_v.append(v, slots)
        assert_pool(cache, of_k, of_v, torch.arange(blocks * bs))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,bs,n", [(2, 64, 1300), (1, 32, 1025), (4, 64, 200)])
def test_rotated_runs(hip, dtype, hkv, bs, n):
    from minillm.attention import get_backend
    from minillm.model.llama import apply_rotary

    rng, g, h = random.Random(n), torch.Generator().manual_seed(n), 2 * hkv
    blocks = 4 * n // bs + 20
    cache, of_k, of_v = filled(rng, g, hkv, blocks, bs, dtype)
    slots = runs(rng, blocks, bs, n, bs)
    n = len(slots)
    qkv = torch.randn(n, h + 2 * hkv, 128, generator=g).to(dtype).to(DEV)
    q, k, v = qkv.split((h, hkv, hkv), dim=1)
    ang = torch.randn(n, 64, generator=g) * 3
    cos, sin = (torch.cat([f(ang)] * 2, dim=1).to(dtype).to(DEV) for f in (torch.cos, torch.sin))
    rot = [apply_rotary(x.transpose(0, 1)[None], cos[None], sin[None])[0].transpose(0, 1).contiguous() for x in (q, k)]

    class Meta(Slots):
        block_size, query_start_loc = bs, [0, n]

    got = get_backend("hip").rope_append(q, k, v, cos, sin, cache.k[0], cache.v[0], Meta(slots.to(DEV)), **cache.scales(0))
    of_k.append(rot[1], slots), of_v.append(v, slots)
    assert torch.equal(bits(got), bits(rot[0]))
    assert_pool(cache, of_k, of_v, torch.arange(blocks * bs))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,bs,n", [(2, 64, 1300), (1, 32, 1025), (4, 64, 200)])
def test_normed_and_rotated_runs(hip, dtype, hkv, bs, n):
    # a key rounds to the 16-bit type (half a step of it) and to e4m3 (2^-4 of that, or half a step of the subnormal grid, 2^-10 of
    # the scale); the fp32 arithmetic before takes 2^-20.  The scale is the one of the largest key of the run or twice it, where
    # that largest key lies within its error of a border.  Values bit for bit
    from minillm.attention import get_backend

    rng, g, h, eps = random.Random(n), torch.Generator().manual_seed(n), 2 * hkv, 1e-5
    blocks = 4 * n // bs + 20
    cache = make_cache(hkv, blocks, bs)
    of_v = PoolByDefinition(blocks, bs, hkv, dtype)
    slots = runs(rng, blocks, bs, n, bs)
    slots = slots[slots >= 0]
    n = len(slots)
    qkv = (torch.randn(n, h + 2 * hkv, 128, generator=g) * torch.logspace(-2, 2, h + 2 * hkv)[:, None]).to(dtype).to(DEV)
    q, k, v = qkv.split((h, hkv, hkv), dim=1)
    wq, wk = ((1 + 0.2 * torch.randn(128, generator=g)).to(dtype).to(DEV) for _ in range(2))
    ang = torch.randn(n, 64, generator=g) * 3
    cos, sin = (torch.cat([f(ang)] * 2, dim=1).to(dtype).to(DEV) for f in (torch.cos, torch.sin))

    class Meta(Slots):
        block_size, query_start_loc = bs, [0, n]

    got = get_backend("hip").rope_append(q, k, v, cos, sin, cache.k[0], cache.v[0], Meta(slots.to(DEV)), qk_norm=(wq, wk, eps),
                                         **cache.scales(0))

    def formula(x, w):
        y = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps) * w.double()
        turn = torch.cat([-y[..., 64:], y[..., :64]], dim=-1)
        c, s = cos.double()[:, None], sin.double()[:, None]
        return y * c + turn * s, (y * c).abs() + (turn * s).abs()

    half = torch.finfo(dtype).eps / 2
    ref, size = formula(q, wq)
    assert ((got.double() - ref).abs() <= half * ref.abs() + 2.0 ** -20 * size + 2.0 ** -25).all()
    ref, size = formula(k, wk)
    off = half * ref.abs() + 2.0 ** -20 * size + 2.0 ** -25
    gk, gv = cache.read(0, slots.to(DEV), dtype)
    page = (slots // bs).to(DEV)
    e = cache.k_scale[0].view(torch.uint8).double()[page] - 127  # [n, Hkv]
    unit = torch.exp2(e)[..., None]
    assert ((gk.double() - ref).abs() <= off + 2.0 ** -4 * (ref.abs() + off) + 2.0 ** -10 * unit).all()
    least, most = (torch.zeros(blocks, hkv, dtype=torch.float64, device=DEV).scatter_reduce_(0, page[:, None].expand(n, hkv), x.amax(-1), "amax")
                   for x in (ref.abs() - off, ref.abs() + off))
    assert (least[page] <= 448 * unit[..., 0]).all()  # nothing saturates
    began = torch.zeros(blocks, dtype=torch.bool, device=DEV)
    began[page[slots.to(DEV) % bs == 0]] = True  # pages whose scale is this run's alone, and no larger than it needs
    assert (2 * most[page] > 448 * unit[..., 0])[began[page]].all()
    of_v.append(v, slots)
    assert same(gv, of_v.values(slots))
