"""Linear layers of 8-bit blocks without a GPU: the torch path against the definition in float64, and refusals."""

import pytest
import torch

from minillm import _native
from minillm.model import fp8
from minillm.model.fp8 import Fp8Linear, quantize_, quantize_blocks, quantize_rows

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.fixture(scope="module", autouse=True)
def library():
    if not _native.LIB_PATH.exists():
        import build_hip

        build_hip.build()


def values(codes, e):
    """codes [..., B] and e8m0 scales [...] -> float64 values."""
    return codes.double() * torch.exp2(e.view(torch.uint8).double() - 127)[..., None]


def nearest_e4m3(y):
    """y (float64, |y| <= 448) to the nearest of e4m3's 253 finite values, a tie to the even code."""
    grid = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
    d = (y.abs()[..., None] - grid).abs()
    near = d == d.amin(-1, keepdim=True)
    even = near.clone()
    even[..., 1::2] = False
    pick = torch.where(even.any(-1), even.double().argmax(-1), near.double().argmax(-1))
    return grid[pick] * torch.sign(y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_are_quantised_by_the_definition(dtype):
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(40, 400, generator=g) * torch.exp(4 * torch.randn(40, 1, generator=g)) * 0.01).to(dtype)
    x[0], x[1, :128], x[2, 5], x[3, 130] = 0, 448.0, 449.0, 448.0
    codes, e = quantize_rows(x)
    assert codes.shape == (40, 512) and e.shape == (40, 4) and codes.dtype == E4M3 and e.dtype == E8M0
    b = torch.nn.functional.pad(x.double(), (0, 112)).view(40, 4, 128)
    s = torch.exp2(e.view(torch.uint8).double() - 127)
    amax = b.abs().amax(-1)
    assert bool((amax <= 448 * s).all()) and bool((amax[amax > 0] > 224 * s[amax > 0]).all())  # the least power of two
    assert torch.equal(values(codes.view(40, 4, 128), e), nearest_e4m3(b / s[..., None]) * s[..., None])


def test_blocks_that_are_not_finite():
    x = torch.ones(3, 256)
    x[1, 3], x[2, 200] = float("inf"), float("nan")
    codes, e = quantize_rows(x)
    assert e.view(torch.uint8)[:, 0].tolist()[1] == 255 and e.view(torch.uint8)[2].tolist()[1] == 255
    y = Fp8Linear.from_linear(torch.nn.Linear(256, 16, bias=False))(x)
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1:]).all()


@pytest.mark.parametrize("n,k", [(16, 16), (272, 400), (128, 128), (48, 1040)])
def test_layer_is_the_product_of_the_quantised_values(n, k):
    torch.manual_seed(n)
    lin = torch.nn.Linear(k, n, bias=False)
    layer = Fp8Linear.from_linear(lin)
    codes, s = quantize_blocks(lin.weight.detach())
    w = codes.double() * torch.exp2(s.view(torch.uint8).double() - 127).repeat_interleave(128, 0)[:n] \
        .repeat_interleave(128, 1)[:, :k]
    assert torch.equal(layer.dequantized().double(), w)
    assert bool(((w - lin.weight.double()).abs() <= 2.0 ** -4 * lin.weight.double().abs() + 2.0 ** -10 * lin.weight.abs().max()).all())
    x = torch.randn(2, 3, k)
    with torch.no_grad():
        y = layer(x)
    c, e = quantize_rows(x.view(6, k))
    v = values(c.view(6, -1, 128), e).flatten(1)[:, :k]
    # fp32 sums of k products: each addition is off by at most 2^-24 of the magnitudes' sum
    bound = k * 2.0 ** -24 * (v.abs() @ w.abs().t()) + 2.0 ** -24 * (v @ w.t()).abs()
    assert bool(((y.view(6, n).double() - v @ w.t()).abs() <= bound).all())
    assert layer(x[:0]).shape == (0, 3, n)


def test_state_round_trip_and_parts():
    layer = Fp8Linear.from_linear(torch.nn.Linear(400, 272, bias=False))
    assert layer.weight.shape == (272, 512) and bool((layer.weight.view(torch.uint8)[:, 400:] == 0).all())
    other = Fp8Linear(400, 272)
    other.load_state_dict(layer.state_dict())
    x = torch.randn(2, 400)
    assert torch.equal(other(x), layer(x)) and "in_features=400" in repr(layer)
    codes = torch.zeros(32, 256).to(E4M3)
    kept = Fp8Linear.from_parts(codes, torch.full((1, 2), 127, dtype=torch.uint8).view(E8M0))
    assert kept.weight.data_ptr() == codes.data_ptr()  # not copied


def test_refusals():
    codes, s = quantize_blocks(torch.randn(32, 256))
    for bad in ((codes.view(torch.uint8), s), (codes[0], s)):
        with pytest.raises(ValueError, match="float8_e4m3fn"):
            Fp8Linear.from_parts(*bad)
    for bad in (s.view(torch.uint8), s[:, :1], s.t()):
        with pytest.raises(ValueError, match="weight_scale"):
            Fp8Linear.from_parts(codes, bad)
    for n, k in ((16, 24), (8, 16), (0, 16)):
        with pytest.raises(ValueError, match="multiples of 16"):
            Fp8Linear(k, n)
    with pytest.raises(ValueError, match="no bias"):
        Fp8Linear.from_linear(torch.nn.Linear(16, 16))
    layer = Fp8Linear.from_parts(codes, s)
    with pytest.raises(ValueError, match="256 columns"):
        layer(torch.randn(3, 128))
    with pytest.raises(RuntimeError, match="inference"):
        layer(torch.randn(3, 256, requires_grad=True))
    with torch.no_grad():
        layer(torch.randn(3, 256, requires_grad=True))


def test_entry_point_checks_its_arguments():
    lib = _native.lib()
    a = 1 << 20  # an aligned address that nothing reads: every call below is refused before its launch

    def call(x=a, stride=256, m=100, k=256, w=a, s=a, n=256, dtype=2, ws=None, size=0, out=a):
        lib.call("mllm_fp8_linear", x, stride, m, k, w, s, n, dtype, ws, size, out, None)

    for kw, match in ((dict(dtype=0), "bfloat16 or float16"), (dict(k=0), "bad sizes"), (dict(m=-1), "bad sizes"),
                      (dict(k=264), "multiples of 16"), (dict(n=250), "multiples of 16"), (dict(k=1 << 24), "too large"),
                      (dict(x=None), "null pointer"), (dict(s=None), "null pointer"), (dict(x=a + 2), "aligned"),
                      (dict(stride=257), "aligned"), (dict(s=a + 1), "aligned"), (dict(), "workspace"),
                      (dict(ws=a + 16, size=1 << 40), "workspace"), (dict(ws=a, size=1), "workspace")):
        with pytest.raises(ValueError, match=match):
            call(**kw)
    call(m=0, x=None, w=None, s=None, out=None)
    need = lib.fn("mllm_fp8_linear_workspace_bytes")
    assert need(0, 256, 256, 256) == 0 and need(16, 4096, 4096, 256) == 0 < need(17, 4096, 4096, 256) < need(65, 4096, 4096, 256)
    assert need(1, 14336, 4096, 256) == 2 * 4 * 14336  # two parts of K, fp32
    assert need(8192, 4096, 4096, 256) >= 8192 * (4096 + 32)


def test_quantize_model():
    from minillm.attention.base import AttentionBackend
    from minillm.model.config import LlamaConfig
    from minillm.model.llama import LlamaForCausalLM, random_init_

    class Causal(AttentionBackend):
        def prefill(self, q, k, v, key_valid=None, **kwargs):
            g = q.shape[1] // k.shape[1]
            return torch.nn.functional.scaled_dot_product_attention(q, k.repeat_interleave(g, 1), v.repeat_interleave(g, 1),
                                                                    is_causal=True)

        def forward(self, *args):
            raise NotImplementedError

    cfg = LlamaConfig(vocab_size=96, hidden_size=64, intermediate_size=144, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=16, rms_norm_eps=1e-5, rope_theta=1e4, qk_norm=True)
    model = random_init_(LlamaForCausalLM(cfg, Causal()))
    assert quantize_(model) is model and quantize_(model) is model  # a second time changes nothing
    kinds = [type(m).__name__ for m in model.modules()]
    assert kinds.count("Fp8Linear") == 14 and kinds.count("Linear") == 1
    with torch.no_grad():
        assert torch.isfinite(model(torch.arange(20)[None])).all()


def test_quantize_changes_all_or_nothing():
    from minillm.model.config import LlamaConfig
    from minillm.model.llama import LlamaForCausalLM

    class NoBackend:
        pass

    cfg = LlamaConfig(vocab_size=32, hidden_size=64, intermediate_size=72, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=16, rms_norm_eps=1e-5, rope_theta=1e4)
    model = LlamaForCausalLM(cfg, NoBackend())
    with pytest.raises(ValueError, match="gate_proj must have"):
        quantize_(model)
    assert not any(isinstance(m, Fp8Linear) for m in model.modules())


def test_casts_leave_codes_and_scales_alone():
    layer = Fp8Linear.from_linear(torch.nn.Linear(272, 48, bias=False))
    codes, scales = layer.weight.view(torch.uint8).clone(), layer.weight_scale.view(torch.uint8).clone()
    x = torch.randn(3, 272)
    want = layer(x)
    for cast in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.to("cpu", torch.float16)):
        stack = cast(torch.nn.Sequential(layer, torch.nn.Linear(48, 2)))
        assert stack[1].weight.dtype != torch.float32
        assert layer.weight.dtype == torch.float8_e4m3fn and layer.weight_scale.dtype == torch.float8_e8m0fnu
        assert torch.equal(layer.weight.view(torch.uint8), codes) and torch.equal(layer.weight_scale.view(torch.uint8), scales)
        assert torch.equal(layer(x), want)
    moved = layer.to("meta")
    assert moved.weight.device.type == "meta" and moved.weight.dtype == torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast_does_not_reach_the_product(dtype):
    layer = Fp8Linear.from_linear(torch.nn.Linear(400, 48, bias=False))
    x = torch.randn(5, 400)
    x[2] *= 1e6  # past fp16's range
    want = layer(x)
    assert torch.isfinite(want).all()
    compiled = torch.compile(layer, fullgraph=True, backend="eager")
    with torch.no_grad(), torch.autocast("cpu", dtype):
        for call in (layer, compiled):
            got = call(x)
            assert got.dtype == x.dtype and torch.equal(got, want)
        assert torch.is_autocast_enabled("cpu") and torch.equal(layer(x[:2].to(dtype)), layer(x[:2].to(dtype).float()).to(dtype))
    assert layer.to("meta")(x.to("meta")).shape == (5, 48)  # a device that has no autocast


def test_every_scale_code_is_its_power_of_two():
    e = torch.arange(256, dtype=torch.uint8)
    want = torch.where(e == 255, float("nan"), torch.exp2(e.double() - 127))
    assert torch.equal(fp8._powers(e).double().nan_to_num(-1.0), want.nan_to_num(-1.0))
    # weights quantised elsewhere under the least scale, and rows large enough for normal sums
    codes = torch.arange(16 * 128, dtype=torch.int32).remainder(127).to(torch.uint8).view(16, 128).view(E4M3)
    layer = Fp8Linear.from_parts(codes, torch.zeros(1, 1, dtype=torch.uint8).view(E8M0))
    assert torch.equal(layer.dequantized().double(), codes.double() * 2.0 ** -127)
    x = torch.full((2, 128), 2.0 ** 90)
    y = layer(x)
    assert bool((y > 0).all()) and torch.equal(y.double(), (x.double() @ (codes.double() * 2.0 ** -127).t()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.bfloat16, "torch.HalfTensor"])
def test_type_leaves_codes_and_scales_alone(dtype):
    layer = Fp8Linear.from_linear(torch.nn.Linear(272, 48, bias=False))
    codes, scales = layer.weight.view(torch.uint8).clone(), layer.weight_scale.view(torch.uint8).clone()
    torch.nn.Sequential(layer, torch.nn.Linear(48, 2)).type(dtype)
    assert layer.weight.dtype == E4M3 and layer.weight_scale.dtype == E8M0
    assert torch.equal(layer.weight.view(torch.uint8), codes) and torch.equal(layer.weight_scale.view(torch.uint8), scales)


def test_quantize_refuses_projections_that_do_more():
    from minillm.model.config import LlamaConfig
    from minillm.model.llama import LlamaForCausalLM

    class NoBackend:
        pass

    class Scaled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    class Named(torch.nn.Linear):
        pass

    def model():
        cfg = LlamaConfig(vocab_size=32, hidden_size=64, intermediate_size=80, num_hidden_layers=2, num_attention_heads=4,
                          num_key_value_heads=2, head_dim=16, rms_norm_eps=1e-5, rope_theta=1e4)
        return LlamaForCausalLM(cfg, NoBackend())

    def own_forward(mlp):
        mlp.up_proj.forward = lambda x: x

    for change in (lambda mlp: setattr(mlp, "up_proj", Scaled(64, 80, bias=False)), own_forward,
                   lambda mlp: mlp.up_proj.register_forward_hook(lambda m, a, y: 2 * y),
                   lambda mlp: mlp.up_proj.register_forward_pre_hook(lambda m, a: a)):
        m = model()
        change(m.model.layers[1].mlp)
        with pytest.raises(ValueError, match="up_proj must be a linear layer without"):
            quantize_(m)
        assert not any(isinstance(x, Fp8Linear) for x in m.modules())
    m = model()  # a subclass that computes the same, and a weight that is computed
    m.model.layers[1].mlp.up_proj = Named(64, 80, bias=False)
    q_proj = m.model.layers[0].self_attn.q_proj
    torch.nn.utils.parametrizations.weight_norm(q_proj)
    want = quantize_blocks(q_proj.weight.detach())[0]
    quantize_(m)
    assert sum(isinstance(x, Fp8Linear) for x in m.modules()) == 14
    assert torch.equal(m.model.layers[0].self_attn.q_proj.weight[:, :64].view(torch.uint8), want.view(torch.uint8))
