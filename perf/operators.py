"""Cases for the operators of a decoder layer served from 4- and 8-bit storage, with a plain form of each in elementary
torch operations, their algorithmic work and a float64 computation of the same outputs.

Operators (the field `op`):
  attend  attention of a step's new tokens over a paged cache held in 4 bits: `HipBackend.attend`.
  append  a step's keys and values into that cache, and its rows read back: `HipBackend.append`, `PagedKVCache.read`.
  norm    RMSNorm of queries and keys for each head with the rotation in the same pass: `HipBackend.rope_append` with
          `qk_norm` (the rotated keys go into the pool), or `kernels.qk_norm_rope` on contiguous tensors (form "rows").
  linear  a product of 8-bit blocks: `Fp8Linear` on 16-bit rows.

The 4-bit format: e2m1 codes, two to a byte (the even dim in the low half), with one power-of-two scale (e8m0) for 32
consecutive dims of a token and head: the least one under which the block's largest magnitude rounds to at most 6.
The 8-bit format: e4m3 codes with one power-of-two scale for 128 columns of a row (activations) or for 128 x 128 weights:
the least one under which the block's largest magnitude is at most 448.  With such scales every quantised value is an
exact function of its block.

Rows of `attend` are (cached tokens, new tokens), from a rule named by `rows` and the case's `shape_seed`, so every
preparation of a case has the same sizes, whatever its values.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False  # true: `run` calls the framework; false: the plain form

DEV = "cuda:0"
BLOCK = 16
DH = 128
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SCALE_RANGE = {torch.bfloat16: (1, 252), torch.float16: (104, 140)}  # e8m0 codes whose values the type holds
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed() -> list[dict]:
    return [
        # four chat requests early in their answers: the smallest step of a server (latency)
        {"name": "kv4_decode_4", "op": "attend", "rows": "decode", "n": 4, "lo": 100, "hi": 700, "shape_seed": 1,
         "dtype": "bf16", "h": 32, "hkv": 8},
        # a full decode step: 256 requests of 128-4096 tokens (the framework's headline workload)
        {"name": "kv4_decode_256", "op": "attend", "rows": "decode", "n": 256, "lo": 128, "hi": 4096, "shape_seed": 2,
         "dtype": "bf16", "h": 32, "hkv": 8},
        # three requests over long documents, on a shard that holds two of the KV heads, in fp16
        {"name": "kv4_decode_long_fp16", "op": "attend", "rows": "decode", "n": 3, "lo": 50000, "hi": 120000,
         "shape_seed": 3, "dtype": "fp16", "h": 16, "hkv": 2},
        # continuous batching under load: prompt chunks admitted beside decode rows
        {"name": "kv4_mixed_48", "op": "attend", "rows": "mixed", "n": 40, "lo": 256, "hi": 8192, "chunks": 8,
         "new": 512, "past": 1024, "shape_seed": 4, "dtype": "bf16", "h": 32, "hkv": 8},
        # prompts of uneven length behind a long common prefix
        {"name": "kv4_prompt_24", "op": "attend", "rows": "mixed", "n": 0, "lo": 1, "hi": 1, "chunks": 24, "new": 700,
         "past": 2048, "shape_seed": 5, "dtype": "bf16", "h": 32, "hkv": 8},
        # the rows of a small decode step
        {"name": "kv4_append_8", "op": "append", "n": 8, "dtype": "bf16", "hkv": 8},
        # the rows of a full prompt step, an odd number of them
        {"name": "kv4_append_8191", "op": "append", "n": 8191, "dtype": "fp16", "hkv": 8},
        # q and k of a decode step, rotated into a 16-bit pool
        {"name": "qk_norm_append_32", "op": "norm", "form": "append", "b": 1, "t": 32, "dtype": "bf16", "h": 32,
         "hkv": 8, "dh": 128},
        # a scored batch of long prompts without a cache
        {"name": "qk_norm_rows_4x2049", "op": "norm", "form": "rows", "b": 4, "t": 2049, "dtype": "bf16", "h": 32,
         "hkv": 8, "dh": 128},
        # the output product of a decode step
        {"name": "fp8_linear_8", "op": "linear", "m": 8, "k": 4096, "n": 4096, "dtype": "bf16"},
        # the gate product of a few short prompts, in fp16
        {"name": "fp8_linear_777_fp16", "op": "linear", "m": 777, "k": 4096, "n": 14336, "dtype": "fp16"},
        # the down product of a full prompt step
        {"name": "fp8_linear_8192", "op": "linear", "m": 8192, "k": 14336, "n": 4096, "dtype": "bf16"},
    ]


def draw(rng: random.Random) -> dict:
    """One more case of the listed ranges: odd sizes, other head counts (a tensor-parallel shard's) and both types."""

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attend", "attend", "attend", "append", "norm", "norm", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "append":
        return {"op": op, "n": log(1, 8192), "dtype": dtype, "hkv": rng.choice([8, 8, 4, 2, 1])}
    if op == "norm":
        h, hkv = rng.choice([(32, 8), (16, 4), (8, 8), (8, 1), (12, 4)])
        form = rng.choice(["append", "rows"])
        b = 1 if form == "append" else rng.choice([1, 2, 3, 4])
        return {"op": op, "form": form, "b": b, "t": log(1, 8192 // b), "dtype": dtype, "h": h, "hkv": hkv,
                "dh": rng.choice([128, 128, 64, 96, 256])}
    if op == "linear":
        k, n = 16 * log(16, 896), 16 * log(8, 896)
        return {"op": op, "m": min(log(1, 8192), max(1, 2 ** 38 // (k * n))), "k": k, "n": n, "dtype": dtype}
    h, hkv = rng.choice([(32, 8), (32, 8), (16, 2), (8, 2), (8, 8), (16, 1)])
    case = {"op": op, "rows": rng.choice(["decode", "decode", "mixed"]), "shape_seed": rng.randrange(1 << 20),
            "dtype": dtype, "h": h, "hkv": hkv}
    if case["rows"] == "decode":
        hi = log(64, 100000)
        case.update(n=max(1, min(log(1, 256), 2 ** 19 // hi)), lo=max(1, hi // 32), hi=hi)
    else:
        hi = log(256, 8192)
        case.update(n=rng.choice([0, log(1, 32)]), lo=max(1, hi // 16), hi=hi, chunks=log(1, 16), new=log(2, 700),
                    past=rng.choice([0, log(1, 2048)]))
    return case


# ---------------------------------------------------------------- sizes


def _rows(case) -> list[tuple[int, int]]:
    """(cached, new) of each sequence of an attend case."""
    r = random.Random(case["shape_seed"])
    rows = [(r.randint(case["lo"], case["hi"]) - 1, 1) for _ in range(case["n"])]
    if case["rows"] == "mixed":  # at least two new tokens: a row with one is a decode row
        rows += [(r.randint(case["past"] // 2, case["past"]), r.randint(max(2, case["new"] // 2), max(2, case["new"])))
                 for _ in range(case["chunks"])]
    return rows


def _visible(rows) -> int:
    """(query, key) pairs of the causal attention."""
    return sum(n * c + n * (n + 1) // 2 for c, n in rows)


def work(case) -> dict:
    if case["op"] == "attend":
        rows = _rows(case)
        tokens, ctx = sum(n for _, n in rows), sum(c + n for c, n in rows)
        kv = 2 * case["hkv"] * (DH // 2 + DH // 32) * ctx
        return {"bytes": kv + 4 * tokens * case["h"] * DH, "flops": 4 * case["h"] * DH * _visible(rows)}
    if case["op"] == "append":  # 16-bit rows in, codes and scales out, and the same codes read back into 16-bit rows
        values = 2 * case["n"] * case["hkv"] * DH
        return {"bytes": 2 * values + 2 * values * 17 // 32 + 2 * values, "flops": 4 * values}
    if case["op"] == "norm":
        tokens = case["b"] * case["t"]
        moved = case["h"] + case["hkv"] * (2 if case["form"] == "append" else 1)
        return {"bytes": 4 * tokens * moved * case["dh"] + 4 * tokens * case["dh"],
                "flops": 8 * tokens * (case["h"] + case["hkv"]) * case["dh"]}
    m, k, n = case["m"], case["k"], case["n"]
    return {"bytes": 2 * m * k + n * k + 2 * m * n, "flops": 2 * m * n * k}


# ---------------------------------------------------------------- the formats, plainly


def _exponent(x: torch.Tensor, carry: int, top: int, lo: int, hi: int) -> torch.Tensor:
    """e8m0 codes of the blocks x [..., block] (fp32): the exponent of the largest magnitude, one up where its mantissa
    carries, less `top`; 255 for a block that holds an infinity or a NaN."""
    amax = x.abs().amax(dim=-1)
    e = ((amax.view(torch.int32) + carry) >> 23) - top
    return torch.where(torch.isfinite(amax), e.clamp(lo, hi), 255)


def _power(e: torch.Tensor) -> torch.Tensor:
    """e8m0 codes (1 .. 255) as fp32 values: 2^(e - 127), 255 as NaN."""
    v = (e.to(torch.int32) << 23).view(torch.float32)
    return torch.where(e == 255, float("nan"), v)


def _codes4(x: torch.Tensor, dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., Dh] fp32 -> e2m1 codes [..., Dh] (uint8) and e8m0 codes [..., Dh / 32] (uint8)."""
    blocks = x.unflatten(-1, (-1, 32))
    e = _exponent(blocks, 1 << 21, 2, *SCALE_RANGE[dtype])
    y = blocks * _power(254 - e.clamp(max=253)).unsqueeze(-1)
    a = y.abs()
    mag = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return (mag + 8 * torch.signbit(y)).flatten(-2).to(torch.uint8), e.to(torch.uint8)


def _values4(codes: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """e2m1 codes [..., Dh] and e8m0 codes [..., Dh / 32] -> fp32 values."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    v = table[codes.int()].unflatten(-1, (-1, 32))
    return (v * _power(e.clamp(min=1)).unsqueeze(-1)).flatten(-2)


def _unpack(packed: torch.Tensor) -> torch.Tensor:
    return torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)


def _codes8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Blocks x [..., block] fp32 -> e4m3 codes and e8m0 codes [...].  Rounded to nearest, ties to even."""
    e = _exponent(x, (1 << 21) - 1, 8, 1, 254)
    return (x * _power(254 - e.clamp(max=253)).unsqueeze(-1)).to(torch.float8_e4m3fn), e.to(torch.uint8)


def _padded(x: torch.Tensor, last: int) -> torch.Tensor:
    return torch.nn.functional.pad(x, (0, last - x.shape[-1]))


# ---------------------------------------------------------------- inputs


def _framework():
    root = Path(__file__).resolve().parent.parent / "mini-llm-inference-server_amd"
    if str(root) not in sys.path:
        sys.path.insert(0, str(root))


def _config(case):
    from minillm.model.config import LlamaConfig

    return LlamaConfig(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=1,
                       num_attention_heads=case.get("h", case["hkv"]), num_key_value_heads=case["hkv"],
                       head_dim=case.get("dh", DH), rms_norm_eps=EPS, rope_theta=500000.0)


def _kv_like(shape, g) -> torch.Tensor:
    """N(0, 1) rows of which some dims are several times larger, as keys have them."""
    x = torch.randn(shape, generator=g, device=DEV)
    loud = torch.rand(shape[-2:], generator=g, device=DEV) < 0.03
    return torch.where(loud, 6 * x, x)


def _pool4(x):
    """Rows x [nb, bs, Hkv, Dh] as a cache of 4 bits holds them: packed codes [nb, bs, Hkv, Dh / 2], scales [nb, bs, Hkv, 4]."""
    codes, e = _codes4(x.float(), x.dtype)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), e


def _group(rows, which, starts, tables):
    """Index tensors of the rows `which` (a decode group or a group of chunks) for the plain form."""
    new = max(rows[i][1] for i in which)
    width = max(len(tables[i]) for i in which)
    pages = torch.tensor([tables[i] + [0] * (width - len(tables[i])) for i in which])
    t = torch.arange(new)
    cached = torch.tensor([rows[i][0] for i in which])
    news = torch.tensor([rows[i][1] for i in which])
    start = torch.tensor([starts[i] for i in which])
    real = t[None, :] < news[:, None]
    tok = torch.where(real, start[:, None] + t[None, :], start[:, None])
    flat = real.flatten().nonzero()[:, 0]
    return {"pages": pages.to(DEV), "pos": (cached[:, None] + torch.minimum(t[None, :], news[:, None] - 1)).to(DEV),
            "len": (cached + news).to(DEV), "tok": tok.to(DEV), "flat": flat.to(DEV), "to": tok.flatten()[flat].to(DEV)}


def prepare(case, seed) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"op": case["op"], "dtype": dtype}
    if own:
        _framework()
    if case["op"] == "attend":
        rows, h, hkv = _rows(case), case["h"], case["hkv"]
        need = [-(-(c + n) // BLOCK) for c, n in rows]
        ids = list(range(sum(need)))
        random.Random(seed).shuffle(ids)
        tables = [[ids.pop() for _ in range(w)] for w in need]
        starts = [sum(n for _, n in rows[:i]) for i in range(len(rows))]
        kv = [_kv_like((sum(need), BLOCK, hkv, DH), g).to(dtype) for _ in range(2)]
        s["q"] = torch.randn((sum(n for _, n in rows), h, DH), generator=g, device=DEV).to(dtype)
        if own:
            from minillm.attention import get_backend
            from minillm.attention.metadata import AttentionMetadata, SeqStep
            from minillm.cache.paged import PagedKVCache

            s["backend"] = get_backend("hip")
            s["meta"] = AttentionMetadata.build([SeqStep(c, n, b) for (c, n), b in zip(rows, tables)], BLOCK, DEV)
            s["cache"] = cache = PagedKVCache(_config(case), sum(need), DEV, torch.float4_e2m1fn_x2)
            every = AttentionMetadata.build([SeqStep(0, BLOCK * sum(need), list(range(sum(need))))], BLOCK, DEV)
            s["backend"].append(*(x.flatten(0, 1) for x in kv), cache.k[0], cache.v[0], every, **cache.scales(0))
        else:
            (s["k"], s["ke"]), (s["v"], s["ve"]) = (_pool4(x) for x in kv)
        groups = [[i for i, (_, n) in enumerate(rows) if (n == 1) == one] for one in (True, False)]
        s["groups"] = [_group(rows, w, starts, tables) for w in groups if w]
    elif case["op"] == "append":
        n, hkv = case["n"], case["hkv"]
        s["k"], s["v"] = _kv_like((n, hkv, DH), g).to(dtype), torch.randn((n, hkv, DH), generator=g, device=DEV).to(dtype)
        if own:
            from minillm.attention import get_backend
            from minillm.attention.metadata import AttentionMetadata, SeqStep
            from minillm.cache.paged import PagedKVCache

            blocks = -(-n // BLOCK)
            ids = list(range(blocks))
            random.Random(seed).shuffle(ids)
            s["backend"] = get_backend("hip")
            s["meta"] = AttentionMetadata.build([SeqStep(0, n, ids)], BLOCK, DEV)
            s["cache"] = PagedKVCache(_config(case), blocks, DEV, torch.float4_e2m1fn_x2)
    elif case["op"] == "norm":
        b, t, h, hkv, dh = (case[x] for x in ("b", "t", "h", "hkv", "dh"))
        # one row of q, k and v of each token side by side, as a joint projection gives them; heads of uneven loudness
        qkv = torch.randn((b, t, h + 2 * hkv, dh), generator=g, device=DEV)
        qkv = (qkv * torch.logspace(-1, 1, h + 2 * hkv, device=DEV)[:, None]).to(dtype)
        s["q"], s["k"], s["v"] = (p.transpose(1, 2) for p in qkv.split((h, hkv, hkv), dim=2))
        s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(dh, generator=g, device=DEV)).to(dtype) for _ in range(2))
        past = int(torch.randint(0, 4096, (1,), generator=g, device=DEV))
        ang = (past + torch.arange(t, device=DEV).double())[:, None] * 500000.0 ** -(
            torch.arange(0, dh, 2, device=DEV).double() / dh)
        ang = torch.cat([ang, ang], dim=-1)[None].expand(b, t, dh)
        s["cos"], s["sin"] = ang.cos().to(dtype), ang.sin().to(dtype)
        s["form"] = case["form"]
        if case["form"] == "append":
            blocks = -(-t // BLOCK)
            ids = list(range(blocks))
            random.Random(seed).shuffle(ids)
            s["slots"] = (torch.tensor(ids, device=DEV)[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)).flatten()[:t]
            s["pools"] = [torch.zeros((blocks, BLOCK, hkv, dh), dtype=dtype, device=DEV) for _ in range(2)]
            if own:
                from minillm.attention import get_backend
                from minillm.attention.metadata import AttentionMetadata, SeqStep

                s["backend"] = get_backend("hip")
                s["meta"] = AttentionMetadata.build([SeqStep(0, t, ids)], BLOCK, DEV)
    else:
        m, k, n = case["m"], case["k"], case["n"]
        # hidden states with a few loud columns; weights whose rows differ in size
        x = torch.randn((m, k), generator=g, device=DEV)
        s["x"] = torch.where(torch.rand(k, generator=g, device=DEV) < 0.01, 20 * x, x).to(dtype)
        kb, nb = -(-k // 128), -(-n // 128)
        w = torch.randn((n, k), generator=g, device=DEV) * k ** -0.5
        w = w * torch.exp(0.5 * torch.randn((n, 1), generator=g, device=DEV))
        w = torch.nn.functional.pad(w, (0, 128 * kb - k, 0, 128 * nb - n))
        codes, e = _codes8(w.view(nb, 128, kb, 128).transpose(1, 2).flatten(2))
        s["w"] = codes.view(nb, kb, 128, 128).view(torch.uint8).transpose(1, 2).reshape(128 * nb, 128 * kb)[:n, :k] \
            .contiguous().view(torch.float8_e4m3fn)
        s["we"] = e  # [nb, kb], e8m0 codes
        if own:
            from minillm.model.fp8 import Fp8Linear

            s["layer"] = Fp8Linear.from_parts(s["w"], s["we"].view(torch.float8_e8m0fnu))
    return s


# ---------------------------------------------------------------- one pass


def run(s):
    with torch.inference_mode():
        if own:
            return _own(s)
        return {"attend": _attend, "append": _append, "norm": _norm, "linear": _linear}[s["op"]](s)


def _own(s):
    if s["op"] == "attend":
        cache = s["cache"]
        out = torch.empty_like(s["q"])
        s["backend"].attend(s["q"], cache.k[0], cache.v[0], s["meta"], out, **cache.scales(0))
        return out
    if s["op"] == "append":
        cache = s["cache"]
        s["backend"].append(s["k"], s["v"], cache.k[0], cache.v[0], s["meta"], **cache.scales(0))
        return cache.read(0, s["meta"].slot_mapping, s["dtype"])
    if s["op"] == "norm":
        if s["form"] == "rows":
            from minillm.model import kernels

            return kernels.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["wq"], s["wk"], EPS)
        q, k, v = (s[x][0].transpose(0, 1) for x in "qkv")
        q = s["backend"].rope_append(q, k, v, s["cos"][0], s["sin"][0], *s["pools"], s["meta"],
                                     qk_norm=(s["wq"], s["wk"], EPS))
        return q, *s["pools"]
    return s["layer"](s["x"])


def _attend(s):
    q = s["q"].float()
    out = torch.empty_like(s["q"])
    for g in s["groups"]:  # decode rows, then rows of several new tokens
        rows, new = g["tok"].shape
        k, v = (_values4(_unpack(s[p][g["pages"]]), s[e][g["pages"]]).flatten(1, 2).transpose(1, 2)
                for p, e in (("k", "ke"), ("v", "ve")))  # [S, Hkv, L, Dh]
        hkv, keys = k.shape[1], k.shape[2]
        qs = q[g["tok"]].unflatten(2, (hkv, -1)).permute(0, 2, 3, 1, 4).reshape(rows, hkv, -1, DH)  # [S, Hkv, G T, Dh]
        at = torch.arange(keys, device=q.device)
        v = torch.where((at < g["len"][:, None])[:, None, :, None], v, 0.0)
        scores = torch.matmul(qs, k.transpose(2, 3)) * DH ** -0.5
        seen = at <= g["pos"][..., None]  # [S, T, L]
        scores = scores.unflatten(2, (-1, new)).masked_fill(~seen[:, None, None], float("-inf"))
        p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
        p = p / p.sum(dim=-1, keepdim=True)
        o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (-1, new)).permute(0, 3, 1, 2, 4)  # [S, T, Hkv, G, Dh]
        out[g["to"]] = o.reshape(rows * new, -1, DH)[g["flat"]].to(out.dtype)
    return out


def _append(s):
    return tuple(_values4(*_codes4(s[x].float(), s["dtype"])).to(s["dtype"]) for x in "kv")


def _norm_rope(x, w, cos, sin, dtype):
    """x [B, heads, T, Dh], cos and sin [B, T, Dh]."""
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w.float()
    half = x.shape[-1] // 2
    turned = torch.cat([-y[..., half:], y[..., :half]], dim=-1)
    return (y * cos.float()[:, None] + turned * sin.float()[:, None]).to(dtype)


def _norm(s):
    q, k = (_norm_rope(s[x], s["w" + x], s["cos"], s["sin"], s["dtype"]) for x in "qk")
    if s["form"] == "rows":
        return q, k
    for pool, rows in zip(s["pools"], (k, s["v"])):
        pool.flatten(0, 1)[s["slots"]] = rows[0].transpose(0, 1)
    return q[0].transpose(0, 1).contiguous(), *s["pools"]


def _linear(s):
    k, n = s["x"].shape[1], s["w"].shape[0]
    kb = s["we"].shape[1]
    codes, e = _codes8(_padded(s["x"].float(), 128 * kb).unflatten(-1, (kb, 128)))
    x = (codes.float() * _power(e)[..., None]).flatten(-2)[:, :k]
    w = s["w"].float() * _power(s["we"]).repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return torch.matmul(x, w.t()).to(s["dtype"])


# ---------------------------------------------------------------- float64


def _two_to(e):
    """2^e in float64, from its bits: a device's pow need not be exact."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_to(x, mantissa, least, most):
    """x (float64) to the nearest value with `mantissa` bits after the point above 2^least, multiples of
    2^(least - mantissa) below; ties to the even multiple; at most `most`."""
    _, e = torch.frexp(x)  # |x| in [2^(e - 1), 2^e)
    step = _two_to((e - 1).clamp(min=least) - mantissa)
    return (torch.round(x / step) * step).clamp(-most, most)


def _least_power(amax, most, closed):
    """The least power of two under which amax is below `most` (`closed`: at most `most`)."""
    _, e = torch.frexp(amax / most)  # amax / most in [2^(e - 1), 2^e)
    p = _two_to(e)
    return torch.where(amax / most == p / 2, p / 2, p) if closed else p


def exact(case, seed):
    with torch.inference_mode():
        s = prepare(case, seed)
        if case["op"] == "attend":
            return _exact_attend(s, case)
        if case["op"] == "append":
            lo, hi = (2.0 ** (c - 127) for c in SCALE_RANGE[s["dtype"]])
            got = []
            for x in (s["k"].double(), s["v"].double()):
                blocks = x.unflatten(-1, (-1, 32))
                scale = _least_power(blocks.abs().amax(dim=-1, keepdim=True), 7.0, False).clamp(lo, hi)
                got.append((_round_to(blocks / scale, 1, 0, 6.0) * scale).flatten(-2))
            return tuple(got)
        if case["op"] == "norm":
            half = case["dh"] // 2
            got = []
            for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
                x, cos, sin = x.double(), s["cos"].double()[:, None], s["sin"].double()[:, None]
                y = x * w.double() / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + EPS)
                got.append(torch.cat([y[..., :half] * cos[..., :half] - y[..., half:] * sin[..., :half],
                                      y[..., half:] * cos[..., half:] + y[..., :half] * sin[..., half:]], dim=-1))
            if case["form"] == "rows":
                return tuple(got)
            pools = [p.double() for p in s["pools"]]
            for p, rows in zip(pools, (got[1], s["v"].double())):
                p.view(-1, case["hkv"], case["dh"]).index_copy_(0, s["slots"], rows[0].transpose(0, 1).contiguous())
            return got[0][0].transpose(0, 1).contiguous(), *pools
        out = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device=DEV)
        for b in range(s["we"].shape[1]):
            x = s["x"][:, 128 * b:128 * b + 128].double()
            scale = _least_power(x.abs().amax(dim=1, keepdim=True), 448.0, True).clamp(2.0 ** -126, 2.0 ** 127)
            x = _round_to(x / scale, 3, -6, 448.0) * scale
            w = s["w"][:, 128 * b:128 * b + 128].double()
            rows = _two_to(s["we"][:, b].long() - 127).repeat_interleave(128)[:case["n"]]
            out += x @ (w * rows[:, None]).t()
        return out


def _exact_attend(s, case):
    table = torch.tensor([*E2M1, *(-v for v in E2M1)], dtype=torch.float64, device=DEV)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    per = case["h"] // case["hkv"]
    for g in s["groups"]:
        for i in range(g["tok"].shape[0]):
            keys = int(g["len"][i])
            ids = g["pages"][i, :-(-keys // BLOCK)]
            kv = []
            for p, e in (("k", "ke"), ("v", "ve")):
                packed = s[p][ids].flatten(0, 1)[:keys].long()
                scale = _two_to(s[e][ids].flatten(0, 1)[:keys].long() - 127).repeat_interleave(32, -1)
                kv.append(torch.stack([table[packed % 16], table[packed // 16]], dim=-1).flatten(-2) * scale)
            mine = int((g["to"] >= g["tok"][i, 0]).logical_and(g["to"] <= g["tok"][i].max()).sum())
            first = int(g["tok"][i, 0])
            seen = torch.arange(keys, device=DEV)[None, :] <= g["pos"][i, :mine, None]
            for h in range(case["hkv"]):
                q = s["q"][first:first + mine, h * per:(h + 1) * per].double()
                scores = (q @ kv[0][:, h].t().contiguous() / math.sqrt(DH)).masked_fill(~seen[:, None], -math.inf)
                out[first:first + mine, h * per:(h + 1) * per] = torch.softmax(scores, dim=-1) @ kv[1][:, h].contiguous()
    return out
