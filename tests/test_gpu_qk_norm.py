"""RMSNorm of query and key heads with the rotation in the same pass (`mllm_qk_norm_rope`, `mllm_qk_norm_rope_kv_append`) against
the formula in float64.

The kernel computes in fp32 and rounds once: an output is off by half a step of itself (half the least subnormal, where it
is smaller) and by its fp32 roundings.  Those are relative to |y_d cos_d| + |y_d' sin_d|: at most 22 for the sum of squares (16
products a lane, up to 6 exchanges), halved by the root, 4 for the division, the sum with eps and rsqrtf, 2 for y, 3 for the
rotation, each 2^-24: below 2^-18 together.
"""

import pytest
import torch

from harness import bits
from test_gpu_fp4 import FP4, make_cache, quantised

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5


def formula(x, w, cos, sin, eps=EPS):
    """x [B, heads, T, Dh], cos and sin [B, T, Dh]: the result and the magnitudes it sums, in float64."""
    x, w, cos, sin = x.double(), w.double(), cos.double()[:, None], sin.double()[:, None]
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    half = x.shape[-1] // 2
    turned = torch.cat([-y[..., half:], y[..., :half]], -1)
    return y * cos + turned * sin, (y * cos).abs() + (turned * sin).abs()


def check(got, x, w, cos, sin, eps=EPS):
    ref, mag = formula(x, w, cos, sin, eps)
    half_step = torch.finfo(got.dtype).eps / 2
    bound = half_step * ref.abs() + 2.0 ** -18 * mag + torch.finfo(got.dtype).tiny * half_step
    worst = ((got.double() - ref).abs() / bound.clamp_min(1e-45)).max().item()
    assert worst <= 1.0, f"error {worst:.3f} of its bound"


def inputs(b, t, h, hkv, dh, dtype, seed=0, past=0):
    """q, k, v as a joint projection gives them, norms and tables."""
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b, t, h + 2 * hkv, dh, generator=g) * torch.logspace(-3, 3, h + 2 * hkv)[:, None]
    q, k, v = (x.transpose(1, 2) for x in qkv.to(dtype).to(DEV).split((h, hkv, hkv), dim=2))
    wq, wk = ((1 + 0.5 * torch.randn(dh, generator=g)).to(dtype).to(DEV) for _ in range(2))
    ang = (past + torch.arange(t).double())[:, None] * 10000.0 ** -(torch.arange(0, dh, 2).double() / dh)
    ang = torch.cat([ang, ang], -1)[None]
    cos, sin = (f().to(dtype).to(DEV).expand(b, t, dh) for f in (ang.cos, ang.sin))
    return q, k, v, cos, sin, wq, wk


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,t,h,hkv,dh", [(1, 1, 32, 8, 128), (2, 37, 4, 4, 64), (3, 5, 6, 2, 96), (1, 333, 8, 1, 256),
                                          (2, 3, 1, 1, 16), (1, 9, 3, 3, 1024), (1, 130, 32, 8, 128), (4, 1, 7, 7, 80)])
def test_rows(hip, b, t, h, hkv, dh, dtype):
    from minillm.model import kernels

    q, k, _, cos, sin, wq, wk = inputs(b, t, h, hkv, dh, dtype, seed=dh + t)
    got_q, got_k = kernels.qk_norm_rope(q, k, cos, sin, wq, wk, EPS)
    assert got_q.shape == q.shape and got_k.shape == k.shape
    check(got_q, q, wq, cos, sin)
    check(got_k, k, wk, cos, sin)
    # the same from contiguous rows, and with an odd order of strides
    for view in (lambda x: x.contiguous(), lambda x: x.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)):
        again = kernels.qk_norm_rope(view(q), view(k), cos.contiguous(), sin.contiguous(), wq, wk, EPS)
        assert torch.equal(bits(again[0]), bits(got_q)) and torch.equal(bits(again[1]), bits(got_k))


def test_zero_rows_and_rows_that_are_not_finite(hip):
    from minillm.model import kernels

    q, k, _, cos, sin, wq, wk = inputs(1, 6, 4, 4, 128, torch.bfloat16)
    q, k = q.contiguous(), k.contiguous()
    want_q, want_k = kernels.qk_norm_rope(q, k, cos, sin, wq, wk, EPS)
    q[0, 1, 2] = 0.0
    q[0, 2, 3, 17] = float("nan")
    k[0, 0, 5, 100] = float("inf")
    got_q, got_k = kernels.qk_norm_rope(q, k, cos, sin, wq, wk, EPS)
    assert bool((got_q[0, 1, 2] == 0).all()) and torch.isnan(got_q[0, 2, 3]).all() and torch.isnan(got_k[0, 0, 5, 36])
    want_q[0, 1, 2], want_q[0, 2, 3], want_k[0, 0, 5] = got_q[0, 1, 2], got_q[0, 2, 3], got_k[0, 0, 5]
    assert torch.equal(bits(got_q), bits(want_q)) and torch.equal(bits(got_k), bits(want_k))


def test_largest_fp16_rows_and_no_eps(hip):
    from minillm.model import kernels

    q, k, _, cos, sin, wq, wk = inputs(1, 4, 2, 2, 256, torch.float16)
    q, k = (torch.full_like(q, 65504.0), torch.full_like(k, 2.0 ** -24))
    got_q, got_k = kernels.qk_norm_rope(q, k, cos, sin, wq, wk, 0.0)
    check(got_q, q, wq, cos, sin, 0.0)
    check(got_k, k, wk, cos, sin, 0.0)


class Slots:
    def __init__(self, slots, n, bs):
        self.slot_mapping, self.query_start_loc, self.block_size = slots, [0, n], bs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,h,hkv,dh,bs", [(1, 32, 8, 128, 16), (45, 8, 2, 64, 32), (200, 12, 4, 192, 16), (19, 5, 5, 128, 16)])
def test_append_into_each_pool(hip, t, h, hkv, dh, bs, dtype):
    """q as the contiguous call gives it; the pools as their own quantization of its rotated k, and of v."""
    from minillm.attention import get_backend
    from minillm.model import kernels

    q, k, v, cos, sin, wq, wk = inputs(1, t, h, hkv, dh, dtype, seed=t, past=1000)
    want_q, want_k = (x[0].transpose(0, 1).contiguous() for x in kernels.qk_norm_rope(q, k, cos, sin, wq, wk, EPS))
    q, k, v = (x[0].transpose(0, 1) for x in (q, k, v))
    blocks = -(-t // bs) + 1
    slots = torch.randperm(blocks * bs, generator=torch.Generator().manual_seed(t))[:t].to(DEV)
    if t > 4:
        slots[2] = -1
    real = slots >= 0
    args = (q, k, v, cos[0], sin[0])
    be, meta, norm = get_backend("hip"), Slots(slots, t, bs), (wq, wk, EPS)

    pools = [torch.zeros(blocks, bs, hkv, dh, dtype=dtype, device=DEV) for _ in range(2)]
    got = be.rope_append(*args, *pools, meta, qk_norm=norm)
    assert torch.equal(bits(got), bits(want_q))
    for pool, rows in zip(pools, (want_k, v)):
        expect = torch.zeros_like(pool)
        expect.flatten(0, 1)[slots[real]] = rows[real]
        assert torch.equal(bits(pool), bits(expect))

    ks, vs = 0.031, 0.27
    pools8 = [p.to(torch.float8_e4m3fn).zero_() for p in pools]
    got = be.rope_append(*args, *pools8, meta, k_scale=ks, v_scale=vs, qk_norm=norm)
    assert torch.equal(bits(got), bits(want_q))
    for pool, rows, s in zip(pools8, (want_k, v), (ks, vs)):
        inv = 1 / torch.tensor(s, dtype=torch.float32)
        expect = (rows.float().cpu() * inv).to(torch.float8_e4m3fn).view(torch.uint8)
        assert torch.equal(pool.view(torch.uint8).flatten(0, 1)[slots[real]].cpu(), expect[real.cpu()])

    cache = make_cache(hkv, blocks, bs, dh=dh)
    got = be.rope_append(*args, cache.k[0], cache.v[0], meta, **cache.scales(0), qk_norm=norm)
    assert torch.equal(bits(got), bits(want_q))
    for values, rows in zip(cache.read(0, slots[real], dtype), (want_k, v)):
        assert torch.equal(values.double().cpu(), quantised(rows[real].contiguous().cpu())[0])


def test_forward_rotary_with_norms_is_append_and_attention(hip):
    from minillm.attention import get_backend
    from minillm.attention.metadata import AttentionMetadata, SeqStep

    rows, tables = [(40, 1), (16, 30), (0, 1)], [[3, 7, 1], [2, 9, 4], [5]]
    meta = AttentionMetadata.build([SeqStep(c, n, t) for (c, n), t in zip(rows, tables)], 16, DEV)
    q, k, v, cos, sin, wq, wk = inputs(1, 32, 32, 8, 128, torch.bfloat16, past=40)
    args = [x[0].transpose(0, 1) for x in (q, k, v)] + [cos[0], sin[0]]
    be, norm = get_backend("hip"), (wq, wk, EPS)
    for cache in (make_cache(8, 10), None):
        if cache is None:
            pools, scales = [torch.zeros(10, 16, 8, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)], {}
        else:
            pools, scales = [cache.k[0], cache.v[0]], cache.scales(0)
        got = be.forward_rotary(*args, *pools, meta, **scales, qk_norm=norm)
        q_rot = be.rope_append(*args, *pools, meta, **scales, qk_norm=norm)
        want = torch.empty_like(got)
        be.attend(q_rot, *pools, meta, want, **scales)
        assert torch.equal(bits(got), bits(want))


def test_operands_that_need_a_gradient_are_refused(hip):
    from minillm.model import kernels

    q, k, _, cos, sin, wq, wk = inputs(1, 3, 4, 2, 64, torch.bfloat16)
    for i in range(4):
        args = [q, k, wq, wk]
        args[i] = args[i].detach().clone().requires_grad_()
        a, b, c, d = args
        with pytest.raises(RuntimeError, match="for inference"):
            kernels.qk_norm_rope(a, b, cos, sin, c, d, EPS)
        with torch.no_grad():
            got = kernels.qk_norm_rope(a, b, cos, sin, c, d, EPS)
        assert all(torch.equal(bits(x), bits(y)) for x, y in zip(got, kernels.qk_norm_rope(q, k, cos, sin, wq, wk, EPS)))
