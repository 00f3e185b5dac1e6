"""Attention over a whole prompt (or a further piece of one) with keys and values in hand, on the tcgen05 tensor cores.

The reference hands the prompt to the model's library attention (models/qwen3/modeling_qwen3.py:228-242); this is the
package's own operator for the same place: causal, grouped heads, dense batches (padded on the right or not) and packed
batches of different lengths.  `decode_attention` and `kv8_attention` take over for the tokens that follow.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .rotary import _head_strides

HEAD_DIM = 128
_status: dict = {}


def _status_word(device: torch.device) -> torch.Tensor:
    st = _status.get(device)
    if st is None:
        st = _status[device] = torch.zeros(1, dtype=torch.int32, device=device)
    return st


def prompt_attention_status(device="cuda") -> int:
    """Synchronise and read the sticky status word of the device's prompt-attention calls (0 = fine)."""
    dev = torch.empty(0, device=device).device
    st = _status.get(dev)
    return 0 if st is None else int(st.item())


def _lengths(x, what: str, n: int, device) -> Optional[torch.Tensor]:
    if x is None:
        return None
    if not isinstance(x, torch.Tensor) or x.dtype != torch.int32 or tuple(x.shape) != (n,) or x.device != device:
        raise ValueError(f"{what} must be an int32 tensor [{n}] on {device}")
    return x.contiguous()


def _source(x: torch.Tensor) -> torch.Tensor:
    """The tensor itself where the copies can read it in place: consecutive channels, no repeated dimension."""
    bad = x.stride(-1) != 1 or any(n > 1 and s <= 0 for n, s in zip(x.shape, x.stride()))
    return x.contiguous() if bad else x


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, scaling: float, *, causal: bool = True,
                     query_lengths: Optional[torch.Tensor] = None, key_lengths: Optional[torch.Tensor] = None,
                     cu_seqlens: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scaling * query key^T) value of every query row, fp16 or bf16, head_dim 128, any group of query heads per
    key head, any strides with consecutive channels.

    Dense: query [B, H_Q, Lq, 128], key / value [B, H, Lk, 128]; query_lengths / key_lengths (int32 [B], on the device)
    for a batch padded on the right.  Returns [B, Lq, H_Q, 128]; padding rows are zeros.
    Packed: query [T, H_Q, 128], key / value [Tk, H, 128], cu_seqlens int32 [N + 1] on the device with sequence s at rows
    cu_seqlens[s] .. cu_seqlens[s + 1] (cu_seqlens_k for the keys where they differ).  Returns [T, H_Q, 128]; rows that
    belong to no sequence behind the last one are zeros in a new tensor and left as they are in a given `out`.

    causal: the last query of a sequence sees its last key, so with more keys than queries the queries are a further
    piece of a prompt.  A row that sees no key is zero.  What a row does not see does not reach it, whatever it holds."""
    packed = cu_seqlens is not None
    dims = 3 if packed else 4
    form = "[T, H, 128]" if packed else "[B, H, T, 128]"
    for x, what in ((query, "query"), (key, "key"), (value, "value")):
        if x.dim() != dims or x.shape[-1] != HEAD_DIM:
            raise ValueError(f"expected {what} {form}, got {tuple(x.shape)}")
        if not x.is_cuda:
            raise ValueError(f"kitty_b200 has no CPU path: the {what} must be on a CUDA device")
        if x.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"prompt_attention takes float16 or bfloat16 tensors, got {x.dtype}")
        if x.dtype != query.dtype or x.device != query.device:
            raise ValueError("query, key and value must agree in type and device")
    if key.shape != value.shape:
        raise ValueError(f"key and value differ in shape: {tuple(key.shape)} and {tuple(value.shape)}")
    dev = query.device
    h_q, h_kv = query.shape[1], key.shape[1]
    if h_kv == 0 or h_q == 0 or h_q % h_kv:
        raise ValueError(f"{h_q} query heads over {h_kv} key heads")
    if not (scaling > 0 and scaling < float("inf")):
        raise ValueError(f"scaling must be positive and finite, got {scaling}")
    if packed:
        if query_lengths is not None or key_lengths is not None:
            raise ValueError("a packed batch takes its lengths from cu_seqlens")
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
            raise ValueError("cu_seqlens must be int32 [N + 1]")
        n = cu_seqlens.shape[0]
        cu_q, cu_k = _lengths(cu_seqlens, "cu_seqlens", n, dev), _lengths(cu_seqlens_k, "cu_seqlens_k", n, dev)
        if cu_k is None and key.shape[0] != query.shape[0]:
            raise ValueError("keys of another number of rows than the queries need cu_seqlens_k")
        B, Lq, Lk = n - 1, query.shape[0], key.shape[0]
        q_len = k_len = None
        shape = (Lq, h_q, HEAD_DIM)
    else:
        if cu_seqlens_k is not None:
            raise ValueError("cu_seqlens_k goes with cu_seqlens")
        B, Lq, Lk = query.shape[0], query.shape[2], key.shape[2]
        if key.shape[0] != B:
            raise ValueError(f"{B} query rows and {key.shape[0]} key rows")
        q_len = _lengths(query_lengths, "query_lengths", B, dev)
        k_len = _lengths(key_lengths, "key_lengths", B, dev)
        cu_q = cu_k = None
        shape = (B, Lq, h_q, HEAD_DIM)
    zero_rest = out is None
    if out is None:
        out = torch.empty(shape, dtype=query.dtype, device=dev)
    elif tuple(out.shape) != shape or out.dtype != query.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {query.dtype} {list(shape)} on {dev}")
    q, k, v = _source(query), _source(key), _source(value)
    order = (lambda x: [0] + [x.stride(i) if x.shape[i] > 1 else 0 for i in (1, 0)]) if packed else _head_strides
    ptr = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    with torch.cuda.device(dev):
        rc = _lib.lib().kitty_prompt_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.dtype_code(q.dtype),
                                          _lib.i64_array(order(q) + order(k) + order(v)), B, Lq, Lk, h_q, h_kv,
                                          float(scaling), int(causal), ptr(q_len), ptr(k_len), ptr(cu_q), ptr(cu_k),
                                          out.data_ptr(), int(zero_rest), _status_word(dev).data_ptr(),
                                          _lib.stream_ptr(dev))
    _lib.check(rc, "kitty_prompt_attn")
    return out
