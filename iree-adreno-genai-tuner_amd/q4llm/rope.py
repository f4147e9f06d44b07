"""RoPE cos/sin tables for LlamaQ4 (the tables of llama_q4.py:184-192), and the frequencies that the
batched operators (ops.rope_rotate, ops.paged_kv_append) form their angles from.

The reference takes its tables from transformers' LlamaRotaryEmbedding. They are computed here
without transformers, with the same fp32 tensor expressions (default RoPE and the Llama-3 frequency
scaling), so the tables are bit-identical (tests/test_rope_runner_cpu.py checks this against transformers
when it is installed). They are load-time host tables shared by every step; the GPU only gathers
rows of them.
"""

import math
from typing import NamedTuple

import torch


class Rope(NamedTuple):
    """Rotary positions of the batched operators (q4_rope in include/q4llm.h): inv_freq [rot_dim / 2] fp32 (the first
    rot_dim dims of a head are rotated), pairs (2i, 2i + 1) if interleaved else (i, i + rot_dim / 2), and the
    factor on cos and sin."""
    inv_freq: torch.Tensor
    interleaved: bool = False
    mscale: float = 1.0

    def to(self, device):
        return self._replace(inv_freq=self.inv_freq.to(device))


def _rope_params(cfg: dict) -> dict:
    rp = dict(cfg.get("rope_parameters") or {})
    rs = cfg.get("rope_scaling") or {}
    rp.update(rs)
    rp.setdefault("rope_theta", cfg.get("rope_theta", 10000.0))
    rp.setdefault("rope_type", rp.get("type", "default") or "default")
    return rp


def inv_freq(cfg: dict) -> torch.Tensor:
    """Inverse frequencies [head_dim / 2] (fp32): base^(-2i/d), then the Llama-3 scaling when
    rope_type == 'llama3' (wavelengths longer than original_ctx / low_freq_factor are divided by
    `factor`, shorter than original_ctx / high_freq_factor kept, the band in between interpolated)."""
    p = _rope_params(cfg)
    hd = cfg.get("head_dim") or cfg["hidden_size"] // cfg["num_attention_heads"]
    base = p["rope_theta"]
    inv = 1.0 / (base ** (torch.arange(0, hd, 2, dtype=torch.int64).to(dtype=torch.float) / hd))
    kind = p["rope_type"]
    if kind == "default":
        return inv
    if kind != "llama3":
        raise NotImplementedError(f"rope_type {kind!r}")
    factor, lo_f, hi_f = p["factor"], p["low_freq_factor"], p["high_freq_factor"]
    old = p["original_max_position_embeddings"]
    lo_wl, hi_wl = old / lo_f, old / hi_f
    wl = 2 * math.pi / inv
    scaled = torch.where(wl > lo_wl, inv / factor, inv)
    smooth = (old / wl - lo_f) / (hi_f - lo_f)
    blended = (1 - smooth) * scaled / factor + smooth * scaled
    medium = ~(wl < hi_wl) * ~(wl > lo_wl)
    return torch.where(medium, blended, scaled)


def rope_tables(cfg: dict, max_ctx: int):
    """(cos, sin), each [max_ctx, head_dim] fp32: angle(pos, i) = pos * inv_freq[i], halves duplicated."""
    inv = inv_freq(cfg)
    pos = torch.arange(max_ctx)[None, None, :].float()
    ang = (inv[None, :, None] @ pos).transpose(1, 2)[0]  # [max_ctx, hd/2], one fp32 product each
    emb = torch.cat((ang, ang), dim=-1)
    return emb.cos() * 1.0, emb.sin() * 1.0


# The keys of a config's scaling that rope_params goes by (some have no effect on a type and are often there all the same).
_ROPE_KEYS = {"rope_type", "type", "rope_theta", "factor", "original_max_position_embeddings", "partial_rotary_factor"}
_SCALING_KEYS = {"default": set(), "linear": set(), "dynamic": set(), "llama3": {"low_freq_factor", "high_freq_factor"},
                 "yarn": {"beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate", "finetuned"}}


def rope_params(cfg: dict, seq_len: int = None, interleaved: bool = False) -> Rope:
    """The Rope of a model config: partial heads (partial_rotary_factor) and the scalings for long contexts
      default, llama3   as inv_freq
      linear            frequencies / factor (position interpolation)
      dynamic           base grown with seq_len past max_position_embeddings (NTK-aware scaling)
      yarn              frequencies of long wavelengths interpolated, those of short ones kept, in between a ramp over
                        the dims from beta_fast to beta_slow turns within the trained length (whole dims unless truncate
                        is false); cos and sin times attention_factor, or m(mscale) / m(mscale_all_dim) where both are
                        given, else m(1), with m(x) = 0.1 x ln(factor) + 1 (Peng et al. 2023)
    on the host; `.to(device)` for the operators. NotImplementedError for other types and for scaling keys that are not
    known here, which might change the frequencies."""
    p = _rope_params(cfg)
    hd = cfg.get("head_dim") or cfg["hidden_size"] // cfg["num_attention_heads"]
    d = int(hd * p.get("partial_rotary_factor", cfg.get("partial_rotary_factor", 1.0)))
    kind = p["rope_type"]
    if kind not in _SCALING_KEYS:
        raise NotImplementedError(f"rope_type {kind!r}")
    unknown = sorted(k for k, x in p.items() if x is not None and k not in _ROPE_KEYS | _SCALING_KEYS[kind])
    if unknown:
        raise NotImplementedError(f"rope_type {kind!r} with {', '.join(unknown)}")
    if kind in ("default", "llama3"):
        return Rope(inv_freq({**cfg, "head_dim": d}), interleaved)
    base, factor = p["rope_theta"], p["factor"]
    exps = torch.arange(0, d, 2, dtype=torch.int64).to(dtype=torch.float) / d
    if kind == "linear":
        return Rope(1.0 / (base ** exps) / factor, interleaved)
    if kind == "dynamic":
        trained = cfg["max_position_embeddings"]
        n = max(seq_len or trained, trained)
        return Rope(1.0 / ((base * ((factor * n / trained) - (factor - 1)) ** (d / (d - 2))) ** exps), interleaved)
    trained = p.get("original_max_position_embeddings") or cfg["max_position_embeddings"]

    def dim_of(turns):  # the dim whose wavelength makes `turns` turns within the trained length
        return d * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = dim_of(p.get("beta_fast") or 32), dim_of(p.get("beta_slow") or 1)
    if p.get("truncate", True):
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, d - 1)
    ramp = ((torch.arange(d // 2, dtype=torch.float) - lo) / (hi - lo if hi != lo else 0.001)).clamp(0, 1)
    inv = 1.0 / (base ** exps)
    mscale = p.get("attention_factor")
    if mscale is None:
        m = lambda x: 0.1 * x * math.log(factor) + 1.0 if factor > 1 else 1.0  # noqa: E731
        one, all_dim = p.get("mscale"), p.get("mscale_all_dim")
        mscale = m(one) / m(all_dim) if one and all_dim else m(1.0)
    return Rope(inv / factor * ramp + inv * (1 - ramp), interleaved, float(mscale))
