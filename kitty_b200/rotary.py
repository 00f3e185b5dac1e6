"""Rotary positions of prompts and tokens.

`RotaryEmbedding` holds what a model's configuration says about its angles (base, how much of the head turns, pair
layout, scaling for long contexts); `apply_rotary` turns the query and key heads of any number of tokens in one launch.
The reference leaves this to its models' element-wise sequence (models/qwen3/modeling_qwen3.py:222-232), whose roundings
`hf_adapter.rope_decode_token` reproduces for a decode token; here angles, sines and cosines are formed in 64 bits and every
output is rounded once.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

HEAD_DIM = 128
ROPE_LAYOUTS = {"half": _lib.ROPE_HALF, "interleaved": _lib.ROPE_INTERLEAVED}


# Fields of a scaling besides rope_type: those it needs, those that it may have.  (rope_theta and partial_rotary_factor are
# the embedding's base and rotary_dim; a linear scaling has no use for the original length.)
_COMMON = {"rope_type", "type", "rope_theta", "partial_rotary_factor"}
_FIELDS = {
    "default": (set(), set()),
    "linear": ({"factor"}, {"original_max_position_embeddings"}),
    "llama3": ({"factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor"}, set()),
    "yarn": ({"factor", "original_max_position_embeddings"}, {"beta_fast", "beta_slow", "attention_factor", "truncate"}),
}


def _scaled_frequencies(rotary_dim: int, base: float, scaling: Optional[dict]):
    """Radians per position of every pair (Python floats) and the factor on cosine and sine, from the fields of a
    transformers configuration's rope parameters."""
    n = rotary_dim // 2
    inv = [base ** (-2.0 * i / rotary_dim) for i in range(n)]
    if scaling is None:
        return inv, 1.0
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _FIELDS:
        raise ValueError(f"rope scaling {kind!r} is not supported ({', '.join(_FIELDS)})")
    needed, optional = _FIELDS[kind]
    missing = sorted(f for f in needed if scaling.get(f) is None)
    if missing:
        raise ValueError(f"rope scaling {kind!r} needs {', '.join(missing)}")
    unknown = sorted(set(scaling) - needed - optional - _COMMON)
    if unknown:
        raise ValueError(f"rope scaling {kind!r} with {', '.join(unknown)} is not supported")
    if kind == "default":
        return inv, 1.0
    factor = float(scaling["factor"])
    if not (factor > 0 and math.isfinite(factor)):
        raise ValueError(f"rope scaling factor must be positive, got {factor}")
    if kind == "linear":
        return [w / factor for w in inv], 1.0
    original = float(scaling["original_max_position_embeddings"])
    if not (original > 0 and math.isfinite(original)):
        raise ValueError(f"original_max_position_embeddings must be positive, got {original}")
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not high > low:
            raise ValueError(f"high_freq_factor must be above low_freq_factor, got {high} and {low}")
        out = []
        for w in inv:       # few turns over the original context: stretched; many: kept; in between: blended
            mix = min(max((original * w / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            out.append(w / factor * (1.0 - mix) + w * mix)
        return out, 1.0
    # yarn: pairs that make beta_fast turns or more over the original context keep their angle, those with beta_slow or
    # fewer are stretched, a ramp over the pair index in between; all sines and cosines are scaled
    if base == 1.0:
        raise ValueError("yarn scaling needs a base other than 1")

    def index(turns):
        return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    # a field that is there but None means its default, as in the configurations
    def given(name, default):
        value = scaling.get(name)
        return default if value is None else float(value)

    first, last = index(given("beta_fast", 32.0)), index(given("beta_slow", 1.0))
    if scaling.get("truncate", True):
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rotary_dim - 1)
    span = last - first if last != first else 0.001
    out = []
    for i, w in enumerate(inv):
        ramp = min(max((i - first) / span, 0.0), 1.0)
        out.append(w / factor * ramp + w * (1.0 - ramp))
    return out, given("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)


class RotaryEmbedding:
    """Angles of a model's rotary positions, kept on a CUDA device.

    head_dim: 128.  base: default 10000.  rotary_dim: channels that turn (even, default all; the rest keep their value).
    layout: 'half' (pair p = channels p and p + rotary_dim/2) or 'interleaved' (channels 2p and 2p + 1).  scaling: None or
    the rope parameters of a transformers configuration, with `rope_type` 'default', 'linear', 'llama3' or 'yarn'.  Their
    `rope_theta` is the base and their `partial_rotary_factor` the part of the head that turns; an argument that says
    otherwise is refused, and so are fields that are not known here."""

    def __init__(self, head_dim: int = HEAD_DIM, base: Optional[float] = None, rotary_dim: Optional[int] = None,
                 layout: str = "half", scaling: Optional[dict] = None, device="cuda"):
        if head_dim != HEAD_DIM:
            raise ValueError(f"kitty_b200 kernels are built for head_dim=128, got {head_dim}")
        theta, part = (None, None) if scaling is None else (scaling.get("rope_theta"), scaling.get("partial_rotary_factor"))
        if theta is not None:
            if base is not None and float(base) != float(theta):
                raise ValueError(f"base is {base}, the rope parameters say rope_theta={theta}")
            base = theta
        if part is not None:
            turned = int(head_dim * float(part))
            if rotary_dim is not None and int(rotary_dim) != turned:
                raise ValueError(f"rotary_dim is {rotary_dim}, the rope parameters say partial_rotary_factor={part}, that is {turned}")
            rotary_dim = turned
        base = 10000.0 if base is None else float(base)
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if rotary_dim < 2 or rotary_dim > head_dim or rotary_dim % 2:
            raise ValueError(f"rotary_dim must be even and in 2 .. {head_dim}, got {rotary_dim}")
        if layout not in ROPE_LAYOUTS:
            raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
        if not (base > 0 and math.isfinite(base)):
            raise ValueError(f"base must be positive, got {base}")
        inv, self.factor = _scaled_frequencies(rotary_dim, base, scaling)
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("kitty_b200 has no CPU path: the angles live on a CUDA device")
        self.head_dim, self.rotary_dim, self.layout, self.base = head_dim, rotary_dim, layout, base
        self.scaling = dict(scaling) if scaling is not None else None
        self.inv_freq = torch.tensor(inv, dtype=torch.float64)                  # radians per position, on the host
        self._turns = torch.tensor([w / (2 * math.pi) for w in inv], dtype=torch.float64, device=dev)
        self.device = self._turns.device
        step = torch.arange(8, dtype=torch.float64)[:, None] * self.inv_freq
        self._steps = torch.stack((torch.cos(step), torch.sin(step)), -1).to(dev).contiguous()
        self._c_plan = _lib.KittyRotaryPlan(self._turns.data_ptr(), self._steps.data_ptr(), self.factor, rotary_dim, ROPE_LAYOUTS[layout], 0)

    def c_plan(self) -> "_lib.KittyRotaryPlan":
        return self._c_plan


def _rotary_input(x: torch.Tensor, what: str, device):
    if x.dim() != 4 or x.shape[3] != HEAD_DIM:
        raise ValueError(f"expected {what} [B, H, T, 128], got {tuple(x.shape)}")
    if x.device != device:
        if not x.is_cuda:
            raise ValueError(f"kitty_b200 has no CPU path: the {what} must be on a CUDA device")
        raise ValueError(f"the angles are on {device}, the {what} on {x.device}")
    return _lib.head_rows(x)


def _rotary_output(out: torch.Tensor, x: torch.Tensor, what: str):
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{what}_out must have the {what}'s shape, type and device")
    rows, strides = _lib.head_rows(out, repeated=False)
    if rows is not out:
        raise ValueError(f"{what}_out needs consecutive channels, rows on 16-byte boundaries and no expanded dimension")
    return out, strides


def apply_rotary(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, rotary: RotaryEmbedding, *,
                 query_out: Optional[torch.Tensor] = None, key_out: Optional[torch.Tensor] = None):
    """Turn query [B, H_Q, T, 128] and key [B, H, T, 128] (any strides with consecutive channels, fp16 / bf16 / fp32) by
    `positions` (int64 [T], [1, T] or [B, T]).  Returns (query, key) turned, in new tensors of the same memory order,
    or in query_out / key_out, which may be query and key themselves (in place).  An output that shares any other memory
    with an input or with the other output is refused."""
    dev = rotary.device
    _lib.refuse_gradients("apply_rotary", query, key, query_out, key_out)
    (q, q_st), (k, k_st) = _rotary_input(query, "query", dev), _rotary_input(key, "key", dev)
    B, h_q, T, _ = q.shape
    Bk, h_kv, Tk, _ = k.shape
    if Bk != B or Tk != T or k.dtype != q.dtype:
        raise ValueError("query and key must agree in batch, tokens and type")
    code = _lib.dtype_code(q.dtype)
    shape = positions.shape
    if len(shape) == 1:
        rows, cols = 1, shape[0]
    elif len(shape) == 2:
        rows, cols = shape
    else:
        rows = cols = -1
    if cols != T or rows not in (1, B):
        raise ValueError(f"expected positions [T], [1, T] or [B, T] for B={B}, T={T}, got {tuple(shape)}")
    if positions.dtype != torch.int64 or positions.device != dev:
        raise ValueError("positions must be int64 on the query's device")
    if T > 1 and positions.stride(-1) != 1:
        positions = positions.contiguous()
    if query_out is None:
        qo = torch.empty_like(q)
        qo_st = q_st if qo.stride() == q.stride() else _lib.head_rows(qo)[1]
    else:
        qo, qo_st = _rotary_output(query_out, query, "query")
    if key_out is None:
        ko = torch.empty_like(k)
        ko_st = k_st if ko.stride() == k.stride() else _lib.head_rows(ko)[1]
    else:
        ko, ko_st = _rotary_output(key_out, key, "key")
    strides = _lib.i64_array(q_st + k_st + qo_st + ko_st)
    _lib.call_on(dev, _lib.lib().kitty_rotary, "kitty_rotary", rotary.c_plan(), q.data_ptr(), k.data_ptr(),
                 positions.data_ptr(), positions.stride(0) if rows > 1 else 0, qo.data_ptr(), ko.data_ptr(), code, B, T,
                 h_q, h_kv, strides)
    for x in (query_out, key_out):
        if x is not None:
            _lib.written(x)
    return qo, ko
