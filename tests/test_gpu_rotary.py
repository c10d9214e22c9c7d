"""GPU parity of the rotation by positions (`mllm_rotary`, `kernels.rotary`) against the formula in float64.

The tolerance counts the roundings: the angle's part of a turn in fp32 (2^-25 of a turn, 2 pi of it as an angle), cos and sin of
it by the hardware (2^-20 of 1), their products and sum in fp32 (3 half steps of 2^-24), and the result to the 16-bit type
(eps / 2, or half the smallest subnormal).  With s = f (|x_a| + |x_b|): eps/2 |out| + 2^-18 s + half a subnormal step."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16]


def formula(x, positions, inv_freq, interleaved, factor):
    """(rotated, bound of the fp32 part's error) of x [B, heads, T, Dh] in float64."""
    rot = 2 * inv_freq.shape[0]
    x = x.double()
    ang = positions[:, None, :, None].double() * inv_freq.double()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out, size = x.clone(), torch.zeros_like(x)
    out[..., a] = factor * (x[..., a] * ang.cos() - x[..., b] * ang.sin())
    out[..., b] = factor * (x[..., b] * ang.cos() + x[..., a] * ang.sin())
    size[..., a] = size[..., b] = abs(factor) * (x[..., a].abs() + x[..., b].abs())
    return out, size


def check(got, x, *args):
    want, size = formula(x, *args)
    fi = torch.finfo(got.dtype)
    bound = fi.eps / 2 * want.abs() + 2.0 ** -18 * size + fi.smallest_normal * fi.eps / 2
    bound = torch.where(size > 0, bound, 0.0)  # what is not rotated is copied
    assert got.shape == x.shape and ((got.double() - want).abs() <= bound * (1 + fi.eps)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("b,t,h,hkv,dh,rot", [
    (1, 1, 32, 8, 128, 128), (1, 33, 8, 1, 128, 64), (4, 257, 12, 4, 64, 64), (2, 5, 3, 3, 96, 24), (3, 700, 8, 8, 256, 64),
    (1, 9000, 4, 2, 128, 128), (2, 4, 2, 1, 40, 6), (1, 3, 1, 1, 2, 2), (1, 7, 2, 2, 1024, 1024), (1, 11, 5, 1, 80, 80),
    (2, 300, 4, 1, 80, 20)])
def test_forms(hip, dtype, interleaved, b, t, h, hkv, dh, rot):
    from minillm.model import kernels

    g = torch.Generator(device=DEV).manual_seed(t + dh)
    qkv = torch.randn((b, t, h + 2 * hkv, dh), generator=g, device=DEV).to(dtype)  # a joint projection's views
    q, k = qkv[:, :, :h].transpose(1, 2), qkv[:, :, h:h + hkv].transpose(1, 2)
    pos = torch.randint(0, 2000000, (b, t), generator=g, device=DEV)
    inv = (10000.0 ** -(torch.arange(0, rot, 2) / rot)).to(DEV)
    got = kernels.rotary(q, k, pos, inv, interleaved=interleaved, factor=1.25)
    for y, x in zip(got, (q, k)):
        check(y, x, pos, inv, interleaved, 1.25)
    if t > 1 and h > 1:  # the operands' order in memory
        assert got[0].transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_and_negative_positions(hip, dtype):
    # the angle is the formula's product in 64 bits up to 2^26 positions within the usual bound
    from minillm.model import kernels

    q = torch.randn(1, 4, 8, 128, device=DEV).to(dtype)
    pos = torch.tensor([[0, 1, -1, -100000, 1 << 20, (1 << 24) + 1, (1 << 31) + 7, 12345678901]], device=DEV)
    inv = (500000.0 ** -(torch.arange(0, 128, 2) / 128)).to(DEV)
    for inter in (True, False):
        for y in kernels.rotary(q, q, pos.clamp(-(1 << 26), 1 << 26), inv, inter):
            check(y, q, pos.clamp(-(1 << 26), 1 << 26), inv, inter, 1.0)
        far, _ = kernels.rotary(q, q, pos, inv, inter)  # 12345678901 rad: 2^-53 of it is 1.4e-6 rad on either side
        want, size = formula(q, pos, inv, inter, 1.0)
        assert ((far.double() - want).abs() <= torch.finfo(dtype).eps * want.abs() + 2.0 ** -14 * size).all()


def test_strides_and_alignment(hip):
    # rows that start off 16 bytes, a last dim that is not dense, expanded positions, tensors of one head
    from minillm.model import kernels

    g = torch.Generator(device=DEV).manual_seed(1)
    inv = (10000.0 ** -(torch.arange(0, 64, 2) / 64)).to(DEV)
    wide = torch.randn((2, 4, 9, 66), generator=g, device=DEV).to(torch.bfloat16)
    pos = torch.arange(9, device=DEV).expand(2, 9)
    for q in (wide[..., 1:65], wide[..., 2:], wide[..., :64], wide.transpose(2, 3)[:, :, :64].transpose(2, 3)):
        for inter in (True, False):
            for y, x in zip(kernels.rotary(q, q[:, :1], pos, inv, inter), (q, q[:, :1])):
                check(y, x, pos, inv, inter, 1.0)
    dilated = torch.randn((1, 2, 3, 128), generator=g, device=DEV).to(torch.bfloat16)[..., ::2]
    check(kernels.rotary(dilated, dilated, pos[:1, :3], inv)[0], dilated, pos[:1, :3], inv, False, 1.0)
    one = torch.randn((1, 1, 5, 64), generator=g, device=DEV).to(torch.bfloat16)
    for y in kernels.rotary(one.expand(1, 3, 5, 64), one, pos[:1, :5], inv):  # heads that share their memory
        check(y, one.expand_as(y), pos[:1, :5], inv, False, 1.0)
    empty = kernels.rotary(wide[:, :, :0, :64], wide[:, :1, :0, :64], pos[:, :0], inv)
    assert empty[0].shape == (2, 4, 0, 64)


def test_nan_and_infinities_stay_in_their_pairs(hip):
    from minillm.model import kernels

    q = torch.randn(1, 2, 3, 64, device=DEV).to(torch.bfloat16)
    q[0, 1, 2, 5], q[0, 0, 0, 63] = float("nan"), float("inf")
    pos, inv = torch.tensor([[3, 4, 5]], device=DEV), (10000.0 ** -(torch.arange(0, 48, 2) / 48)).to(DEV)
    out, _ = kernels.rotary(q, q, pos, inv)
    bad = ~torch.isfinite(out)
    assert bad.nonzero().tolist() == [[0, 0, 0, 63], [0, 1, 2, 5], [0, 1, 2, 29]]


def test_other_stream_and_captured(hip):
    from minillm.model import kernels

    q = torch.randn(1, 8, 50, 128, device=DEV).to(torch.bfloat16)
    k, pos = q[:, :2].clone(), torch.arange(50, device=DEV)[None] + 7
    inv = (10000.0 ** -(torch.arange(0, 128, 2) / 128)).to(DEV)
    want = kernels.rotary(q, k, pos, inv, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.rotary(q, k, pos, inv, True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.rotary(q, k, pos, inv, True)
    for i in range(3):
        q.copy_(torch.randn(q.shape, device=DEV))
        pos.add_(100 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, kernels.rotary(q, k, pos, inv, True)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_scaled_tables(hip, dtype):
    # half a step of the type, and 2^-18 before it: the part of a turn in fp32 and the hardware's cos and sin
    from minillm.model import kernels

    g = torch.Generator(device=DEV).manual_seed(4)
    pos = torch.randint(-(1 << 22), 1 << 22, (3, 700), generator=g, device=DEV)
    inv = (500000.0 ** -(torch.arange(0, 128, 2) / 128)).to(DEV)
    for got, f in zip(kernels.rope_table(pos, inv, dtype, 1.3), (torch.cos, torch.sin)):
        ang = pos[..., None].double() * inv.double()
        want = 1.3 * f(torch.cat([ang, ang], -1))
        fi = torch.finfo(dtype)
        assert ((got.double() - want).abs() <= fi.eps / 2 * want.abs() + 2.0 ** -18).all()


def test_gradients_are_refused(hip):
    from minillm.model import kernels

    q = torch.randn(1, 2, 3, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    pos, inv = torch.zeros(1, 3, dtype=torch.int64, device=DEV), torch.ones(32, device=DEV)
    with pytest.raises(RuntimeError, match="no gradient"):
        kernels.rotary(q, q, pos, inv)
    with torch.no_grad():
        kernels.rotary(q, q, pos, inv)


@pytest.mark.parametrize("kw", [dict(rope_interleaved=True), dict(partial_rotary_factor=0.5, rope_interleaved=True),
                                dict(rope_scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}),
                                dict(rope_scaling={"rope_type": "linear", "factor": 4.0}, partial_rotary_factor=0.25, qk_norm=True)])
def test_model_forward_and_gradients(hip, kw):
    # the contiguous model on the GPU in bf16 against itself in float32 on the CPU (bf16 activations: 2^-8 of them a layer's
    # few dozen roundings over, and logits of order 1), and with gradients on, where the rotation runs in torch operations
    from minillm.attention import get_backend
    from minillm.model.config import LlamaConfig
    from minillm.model.llama import LlamaForCausalLM, random_init_
    from oracle_engine import OracleBackend

    cfg = LlamaConfig(vocab_size=128, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, rms_norm_eps=1e-5, rope_theta=10000.0, **kw)
    cpu = random_init_(LlamaForCausalLM(cfg, OracleBackend()), std=0.05, seed=2)
    gpu = LlamaForCausalLM(cfg, get_backend("hip")).to(DEV, torch.bfloat16)
    gpu.load_state_dict(cpu.state_dict())
    cpu.load_state_dict({n: p.float().cpu() for n, p in gpu.state_dict().items()})  # the same rounded weights
    ids = torch.randint(0, 128, (2, 70), generator=torch.Generator().manual_seed(3))
    with torch.no_grad():
        want = cpu(ids)
        got = gpu(ids.to(DEV)).float().cpu()
    scale = want.abs().max()
    assert (got - want).abs().max() <= 0.04 * scale
    gpu.set_backend(OracleBackend())
    gpu(ids.to(DEV)).float().square().mean().backward()
    grad = gpu.model.layers[0].self_attn.q_proj.weight.grad
    assert torch.isfinite(grad).all() and grad.abs().max() > 0
