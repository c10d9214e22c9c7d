"""Llama model configuration (reference src/minillm/model/config.py:11-67).

The fields carry the names of Hugging Face `config.json` keys.  `from_dict` reads both the flat layout
(`rope_theta`, `rope_scaling`) and the nested one newer transformers write (`rope_parameters`).
"""

from __future__ import annotations

import json
from collections.abc import Mapping
from dataclasses import dataclass, field
from pathlib import Path
from typing import Any

# keys every config.json must hold, and the optional ones with the value taken when they are absent
_REQUIRED_KEYS = ("vocab_size", "hidden_size", "intermediate_size", "num_hidden_layers", "num_attention_heads",
                  "rms_norm_eps")
_DEFAULTS = {"tie_word_embeddings": False, "max_position_embeddings": 8192, "qk_norm": False}


def _rope_fields(d: Mapping[str, Any]) -> tuple[float, dict[str, Any] | None]:
    """(rope_theta, rope_scaling) of a config dictionary.

    theta: `rope_parameters.rope_theta`, else the top-level `rope_theta`, else 10000.  Scaling: the
    top-level `rope_scaling` entry when it is non-empty, else `rope_parameters` when that names a type
    other than "default".  The type is read from `rope_type`, or from the older `type` key when
    `rope_type` is absent, and stored under `rope_type`; a chosen entry of type "default" or of no type
    means plain RoPE (None).
    """
    nested = d.get("rope_parameters") or {}
    theta = float(nested["rope_theta"] if "rope_theta" in nested else d.get("rope_theta", 10000.0))
    if d.get("rope_scaling"):
        entry = d["rope_scaling"]
    elif nested.get("rope_type", "default") != "default":
        entry = nested
    else:
        return theta, None
    kind = entry["rope_type"] if "rope_type" in entry else entry.get("type")
    if kind is None or kind == "default":
        return theta, None
    return theta, {**entry, "rope_type": kind}


def _eos_ids(value: Any) -> tuple[int, ...]:
    """`eos_token_id` may be absent, one id or a list of ids."""
    if value is None:
        return ()
    if isinstance(value, (list, tuple)):
        return tuple(int(v) for v in value)
    return (int(value),)


@dataclass(frozen=True)
class LlamaConfig:
    vocab_size: int
    hidden_size: int
    intermediate_size: int
    num_hidden_layers: int
    num_attention_heads: int
    num_key_value_heads: int
    head_dim: int
    rms_norm_eps: float
    rope_theta: float
    rope_scaling: dict[str, Any] | None = None  # llama3 frequency scaling, or None for plain RoPE
    tie_word_embeddings: bool = False
    max_position_embeddings: int = 8192
    eos_token_ids: tuple[int, ...] = field(default_factory=tuple)
    qk_norm: bool = False  # RMSNorm of every query and key head before the rotation

    @property
    def num_kv_groups(self) -> int:
        """Query heads per KV head."""
        return self.num_attention_heads // self.num_key_value_heads

    @classmethod
    def from_dict(cls, d: Mapping[str, Any]) -> LlamaConfig:
        """A config.json dictionary -> LlamaConfig; a missing required key raises KeyError."""
        absent = [k for k in _REQUIRED_KEYS if k not in d]
        if absent:
            raise KeyError(f"config.json lacks {', '.join(absent)}")
        kw: dict[str, Any] = {k: d[k] for k in _REQUIRED_KEYS}
        kw.update((k, d.get(k, default)) for k, default in _DEFAULTS.items())
        heads = kw["num_attention_heads"]
        kw["num_key_value_heads"] = d.get("num_key_value_heads", heads)  # absent: one KV head per query head
        kw["head_dim"] = d.get("head_dim") or kw["hidden_size"] // heads
        kw["rope_theta"], kw["rope_scaling"] = _rope_fields(d)
        kw["eos_token_ids"] = _eos_ids(d.get("eos_token_id"))
        return cls(**kw)

    @classmethod
    def from_pretrained(cls, model_dir: str | Path) -> LlamaConfig:
        return cls.from_dict(json.loads((Path(model_dir) / "config.json").read_text()))


LLAMA_3_1_8B = dict(vocab_size=128256, hidden_size=4096, intermediate_size=14336, num_hidden_layers=32,
                    num_attention_heads=32, num_key_value_heads=8, head_dim=128, rms_norm_eps=1e-5,
                    rope_theta=500000.0, max_position_embeddings=131072,
                    rope_scaling={"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                  "high_freq_factor": 4.0, "original_max_position_embeddings": 8192})
