"""Linear layers of 8-bit blocks (`mllm_fp8_linear`, `Fp8Linear`) against the definition in float64.

The quantisation is exact, so the codes and scales of x are the definition's.  What differs is the sum.  The matrix
instruction adds products in groups of eight consecutive k: it aligns them to the largest of the group and drops what lies more
than 13 binary places below that one's power of two (measured: beside a product 2^16 in its group 2^3 survives and 2^2 does
not; beside one in another group every product does).  The largest loses nothing, so a group is off by less than
7 * 2^-13 of its largest product, and that is at most the product of the group's largest |x| and |w|.  Groups and the
accumulator are added with 24 bits: K / 8 additions, 8 of wavefronts or parts of K and one more, each off by at most 2^-23 of the
sum of the magnitudes.  The output is off by half a step of itself besides.
"""

import pytest
import torch

from harness import bits

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantised(x):
    """The float64 values of x's blocks of 128 columns, by the definition."""
    m, k = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -k % 128)).view(m, -1, 128)
    amax = b.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(amax / 448)
    e = torch.where(amax / 448 == two_to(e - 1), e - 1, e).clamp(-126, 127)
    y = b / two_to(e)
    _, t = torch.frexp(y)
    step = two_to((t - 1).clamp(min=-6) - 3)
    v = torch.round(y / step) * step * two_to(e)
    bad = ~torch.isfinite(b).all(-1, keepdim=True)
    return torch.where(bad, float("nan"), v).flatten(1)[:, :k]


def layer(n, k, seed=0, spread=2.0):
    from minillm.model.fp8 import Fp8Linear

    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k), generator=g, dtype=torch.uint8)
    codes = torch.where((codes & 127) == 127, 3, codes)  # no NaN
    scales = (127 - 12 + spread * torch.randn(-(-n // 128), -(-k // 128), generator=g)).round().clamp(1, 254).to(torch.uint8)
    w = codes.view(E4M3).double() * two_to(scales.long() - 127).repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return Fp8Linear.from_parts(codes.view(E4M3).to(DEV), scales.view(E8M0).to(DEV)), w


def rows(m, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 1)
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g)) * torch.exp(torch.randn(m, 1, generator=g))
    return x.clamp(-6e4, 6e4).to(dtype)


def check(got, x, w):
    v = quantised(x).to(DEV)
    w = w.to(DEV)
    ref, mag = v @ w.t(), v.abs() @ w.abs().t()
    k = x.shape[1]
    top_x, top_w = (t.abs().unflatten(1, (k // 8, 8)).amax(-1) for t in (v, w))
    bound = torch.finfo(got.dtype).eps / 2 * ref.abs() + 7 * 2.0 ** -13 * (top_x @ top_w.t()) + (k / 8 + 9) * 2.0 ** -23 * mag
    bound = bound + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    worst = ((got.double() - ref).abs() / bound).max().item()
    assert worst <= 1.0, f"error {worst:.3f} of its bound"


SHAPES = [(1, 128, 16), (1, 4096, 4096), (3, 16, 48), (8, 4096, 1024), (16, 144, 80), (17, 1040, 272), (33, 2048, 112),
          (64, 14336, 4096), (64, 256, 14336), (8, 14336, 4096), (9, 2064, 9216), (32, 5008, 4112),
          (8, 2064, 14336), (16, 4096, 14352), (30, 1168, 16400), (3, 1296, 13200)]
MANY = [(65, 128, 16), (65, 4096, 4096), (100, 144, 272), (129, 2048, 96), (255, 1040, 128), (300, 512, 4096),
        (777, 4096, 1040), (2048, 272, 14336), (4100, 1024, 4112)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", SHAPES + MANY)
def test_shapes(hip, m, k, n, dtype):
    lin, w = layer(n, k, seed=m + k)
    x = rows(m, k, dtype, seed=n)
    with torch.no_grad():
        got = lin(x.to(DEV))
    assert got.shape == (m, n) and got.dtype == dtype
    check(got, x, w)


@pytest.mark.parametrize("m", [5, 64, 200])
def test_quantisation_is_the_definitions(hip, m):
    # identity-like weights (one code 1.0 per row) give back the quantised x itself: every 16-bit pattern's neighbourhood
    from minillm.model.fp8 import Fp8Linear, quantize_rows

    k = 256
    codes = torch.zeros(k, k)
    codes.fill_diagonal_(1.0)
    lin = Fp8Linear.from_parts(codes.to(E4M3).to(DEV), torch.full((2, 2), 127, dtype=torch.uint8).view(E8M0).to(DEV))
    for dtype in (torch.bfloat16, torch.float16):
        pat = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).view(-1, k)
        mix = pat.flatten()[torch.randperm(65536, generator=torch.Generator().manual_seed(m))].view(-1, k)
        x = torch.cat([pat, torch.where(torch.isfinite(mix), mix, 1.0)])
        x = torch.where(x.float().abs() < 2.0 ** 100, x, x * 0.5)  # the largest bf16 values are their own products with zeros
        fine = torch.isfinite(x).view(-1, 2, 128).all(-1).repeat_interleave(128, 1) & torch.isfinite(x).all(-1, keepdim=True)
        with torch.no_grad():
            got = torch.cat([lin(x[i:i + m].to(DEV)) for i in range(0, x.shape[0], m)]).cpu()
        want = quantised(x)
        assert torch.equal(got.double()[fine], want.to(dtype).double()[fine])
        assert torch.isnan(got[~torch.isfinite(x).all(-1)]).all()  # a row that holds an infinity or a NaN
        c, e = quantize_rows(x)
        v = (c.double().view(-1, 2, 128) * two_to(e.view(torch.uint8).long() - 127)[..., None]).flatten(1)
        assert torch.equal(v[fine], want[fine])


@pytest.mark.parametrize("n,k", [(1040, 4096), (8272, 2320), (4096, 4224), (16, 640), (33 * 1024, 1024), (14352, 2320)])
def test_rows_do_not_depend_on_their_batch(hip, n, k):
    lin, _ = layer(n, k)
    x = rows(64, k, torch.bfloat16).to(DEV)
    with torch.no_grad():
        every = lin(x)
        for m in (1, 15, 16, 31, 50):
            assert torch.equal(bits(lin(x[:m])), bits(every[:m]))
            assert torch.equal(bits(lin(x[m:m + 1])), bits(every[m:m + 1]))


@pytest.mark.parametrize("m", [4, 130])
def test_strided_and_shaped_inputs(hip, m):
    lin, _ = layer(272, 512)
    wide = rows(m, 1040, torch.bfloat16).to(DEV)
    with torch.no_grad():
        want = lin(wide[:, 8:520].contiguous())
        assert torch.equal(bits(lin(wide[:, 8:520])), bits(want))  # aligned rows of a wider tensor
        assert torch.equal(bits(lin(wide[:, 8:520].contiguous().view(2, m // 2, 512)).view(m, 272)), bits(want))
        x = wide[:, 3:515]  # rows that are not aligned
        assert torch.equal(bits(lin(x)), bits(lin(x.clone())))
        assert torch.equal(bits(lin(wide[:, 8:520].t().contiguous().t())), bits(want))
        assert lin(wide[:0, 8:520]).shape == (0, 272) and lin(wide[:0, 8:520].view(3, 0, 512)).shape == (3, 0, 272)


def test_nan_weights_and_scales_stay_in_their_outputs(hip):
    from minillm.model.fp8 import Fp8Linear

    for m in (3, 100):
        lin, w = layer(256, 384)
        codes, scales = lin.weight.view(torch.uint8).clone(), lin.weight_scale.view(torch.uint8).clone()
        codes[7, 200] = 127
        scales[1, 2] = 255
        bad = Fp8Linear.from_parts(codes.view(E4M3), scales.view(E8M0))
        x = rows(m, 384, torch.bfloat16).to(DEV)
        with torch.no_grad():
            want, got = lin(x), bad(x)
        assert torch.isnan(got[:, 7]).all() and torch.isnan(got[:, 128:]).all()
        keep = [i for i in range(128) if i != 7]
        assert torch.equal(bits(got[:, keep]), bits(want[:, keep]))


@pytest.mark.parametrize("n,k,sizes", [(1040, 1024, (8, 300)), (9232, 2048, (8, 40)), (1040, 2048, (20, 70))])
def test_captured_calls(hip, n, k, sizes):
    # two graphs of one layer, replayed between eager calls of other sizes
    lin, _ = layer(n, k)
    xs = [rows(m, k, torch.bfloat16, seed=m).to(DEV) for m in sizes]
    graphs = []
    with torch.no_grad():
        want = [lin(x) for x in xs]
        for x in xs:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                lin(x)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = lin(x)
            graphs.append((g, y))
        for _ in range(3):
            for (g, y), w in zip(graphs, want):
                y.zero_()
                g.replay()
                lin(xs[1][:2 * sizes[1] // 3])
                torch.cuda.synchronize()
                assert torch.equal(bits(y), bits(w))


def test_two_streams_at_once(hip):
    lin, _ = layer(9232, 2048)
    xs = [rows(m, 2048, torch.bfloat16, seed=m).to(DEV) for m in (40, 60, 500)]
    streams = [torch.cuda.Stream() for _ in xs]
    with torch.no_grad():
        want = [lin(x) for x in xs]
        torch.cuda.synchronize()
        got = [[], [], []]
        for _ in range(5):
            for x, s, y in zip(xs, streams, got):
                with torch.cuda.stream(s):
                    y.append(lin(x))
        torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(bits(y), bits(w)) for y in ys)


def test_model_of_8bit_blocks(hip):
    """quantize_ on a small model: the layers' outputs are those of the same model in torch operations, within the 16-bit
    roundings between them."""
    from minillm.model.config import LlamaConfig
    from minillm.model.fp8 import Fp8Linear, quantize_
    from minillm.model.llama import LlamaForCausalLM, random_init_

    cfg = LlamaConfig(vocab_size=320, hidden_size=256, intermediate_size=528, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, rms_norm_eps=1e-5, rope_theta=1e4)
    model = quantize_(random_init_(LlamaForCausalLM(cfg).to(device=DEV, dtype=torch.bfloat16)))
    attn, mlp = model.model.layers[1].self_attn, model.model.layers[1].mlp
    assert all(isinstance(m, Fp8Linear) for m in (attn.q_proj, attn.k_proj, attn.v_proj, attn.o_proj, mlp.gate_proj,
                                                  mlp.up_proj, mlp.down_proj))
    assert isinstance(model.lm_head, torch.nn.Linear)
    for t in (9, 100):
        x = torch.randn(1, t, 256, generator=torch.Generator().manual_seed(t)).bfloat16().to(DEV)
        with torch.no_grad():
            got = mlp(x)
            gate, up = mlp.gate_proj(x), mlp.up_proj(x)
            h = (torch.nn.functional.silu(gate.double()) * up.double()).bfloat16()
            assert torch.equal(bits(got), bits(mlp.down_proj(h)))
            ids = torch.randint(0, 320, (1, t), generator=torch.Generator().manual_seed(t)).to(DEV)
            assert torch.isfinite(model(ids)).all()


def check32(got, x, w):
    """The product in torch operations, float32: k additions, each off by at most 2^-24 of the sum of the magnitudes."""
    v = quantised(x)
    want = v @ w.t()
    bound = x.shape[1] * 2.0 ** -24 * (v.abs() @ w.abs().t()) + 2.0 ** -24 * want.abs()
    assert bool(((got.double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("m", [3, 20, 100, 300])
def test_the_least_scale(hip, m):
    # scale code 0 is 2^-127 in each product form and in torch operations on the GPU
    lin, w = layer(4112 if m == 300 else 272, 400, seed=m)
    scales = lin.weight_scale.view(torch.uint8)
    before = scales[0].clone()
    scales[0] = 0
    w[:128] *= two_to(-before.long().cpu()).repeat_interleave(128)[:400]  # 2^(before - 127) to 2^-127
    x = (rows(m, 400, torch.float32, seed=m) * 2.0 ** 100).bfloat16()
    with torch.no_grad():
        got = lin(x.to(DEV))
        assert bool((got[:, :128] != 0).any())
        check(got, x, w)
        check32(lin(x.float().to(DEV)), x, w)


def test_autocast_keeps_the_definition(hip):
    lin, w = layer(272, 400, seed=5)
    x = rows(20, 400, torch.float32, seed=6)
    for dtype in (torch.bfloat16, torch.float16):
        with torch.no_grad(), torch.autocast("cuda", dtype):
            got = lin(x.to(DEV))
        assert got.dtype == x.dtype
        check32(got, x, w)
