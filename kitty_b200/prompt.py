"""Attention over a whole prompt (or a further piece of one) with keys and values in hand, on the tcgen05 tensor cores.

The reference hands the prompt to the model's library attention (models/qwen3/modeling_qwen3.py:228-242); this is the
package's own operator for the same place: causal, grouped heads, dense batches (padded on the right or not) and packed
batches of different lengths.  `decode_attention` and `kv8_attention` take over for the tokens that follow.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _lib

HEAD_DIM = 128
_status: dict = {}


def _status_word(device: torch.device) -> Optional[int]:
    """Address of the device's status word; none during a capture that comes before the device's first call (memory of
    a graph's own pool must not outlive it)."""
    st = _status.get(device)
    if st is None:
        if torch.cuda.is_current_stream_capturing():
            return None
        st = _status.setdefault(device, torch.zeros(1, dtype=torch.int32, device=device))
    return st.data_ptr()


@functools.lru_cache(maxsize=4096)
def _workspace_need(device, B: int, Lq: int, Lk: int, h_q: int, h_kv: int, causal: bool, packed: bool) -> int:
    with torch.cuda.device(device):                     # the plan depends on the device's multiprocessors
        need = _lib.lib().kitty_prompt_workspace_bytes(B, Lq, Lk, h_q, h_kv, int(causal), int(packed))
    if need < 0:
        _lib.check(int(need), "kitty_prompt_workspace_bytes")
    return int(need)


def prompt_attention_status(device="cuda") -> int:
    """Synchronise and read the sticky status word of the device's prompt-attention calls (0 = fine)."""
    dev = torch.empty(0, device=device).device
    st = _status.get(dev)
    return 0 if st is None else int(st.item())


def check_prompt_attention() -> None:
    """Synchronise and raise if a wait has run out in a prompt-attention call of any device (its output is not complete)."""
    for dev, st in list(_status.items()):
        if int(st.item()):
            raise _lib.KittyError(_lib.KITTY_E_TIMEOUT, f"prompt_attention on {dev}")


def _lengths(x, what: str, n: int, device) -> Optional[torch.Tensor]:
    if x is None:
        return None
    if not isinstance(x, torch.Tensor) or x.dtype != torch.int32 or x.shape != (n,) or x.device != device:
        raise ValueError(f"{what} must be an int32 tensor [{n}] on {device}")
    return x.contiguous()


def _source(x: torch.Tensor, what: str, like: torch.Tensor, packed: bool):
    """The tensor as the copies can read it, and its strides."""
    shape, dev = x.shape, x.device
    if len(shape) != (3 if packed else 4) or shape[-1] != HEAD_DIM:
        raise ValueError(f"expected {what} {'[T, H, 128]' if packed else '[B, H, T, 128]'}, got {tuple(shape)}")
    if dev.type != "cuda":
        raise ValueError(f"kitty_b200 has no CPU path: the {what} must be on a CUDA device")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"prompt_attention takes float16 or bfloat16 tensors, got {x.dtype}")
    if x is not like and (x.dtype != like.dtype or dev != like.device):
        raise ValueError("query, key and value must agree in type and device")
    return _lib.head_rows(x, repeated=False)


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, scaling: float, *, causal: bool = True,
                     query_lengths: Optional[torch.Tensor] = None, key_lengths: Optional[torch.Tensor] = None,
                     cu_seqlens: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scaling * query key^T) value of every query row, fp16 or bf16, head_dim 128, any group of query heads per
    key head, any strides with consecutive channels.

    Dense: query [B, H_Q, Lq, 128], key / value [B, H, Lk, 128]; query_lengths / key_lengths (int32 [B], on the device)
    for a batch padded on the right.  Returns [B, Lq, H_Q, 128]; padding rows are zeros.
    Packed: query [T, H_Q, 128], key / value [Tk, H, 128], cu_seqlens int32 [N + 1] on the device, 0 first and never
    falling, with sequence s at rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 (cu_seqlens_k for the keys where they differ).  Returns [T, H_Q, 128]; rows that
    belong to no sequence behind the last one are zeros in a new tensor and left as they are in a given `out`.  An `out`
    that shares memory with an input is refused.

    causal: the last query of a sequence sees its last key, so with more keys than queries the queries are a further
    piece of a prompt.  A row that sees no key is zero.  What a row does not see does not reach it, whatever it holds.

    Weights are rounded to the inputs' type for the product with the values; over very many keys the tensor cores'
    additions cost up to about 2^-26 of a result per key (0.1 % at 65536)."""
    packed = cu_seqlens is not None
    _lib.refuse_gradients("prompt_attention", query, key, value, out)
    q, q_st = _source(query, "query", query, packed)
    k, k_st = _source(key, "key", query, packed)
    v, v_st = _source(value, "value", query, packed)
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
        out = _lib.empty(shape, query.dtype, dev)
    elif tuple(out.shape) != shape or out.dtype != query.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {query.dtype} {list(shape)} on {dev}")
    need = _workspace_need(dev, B, Lq, Lk, h_q, h_kv, bool(causal), packed)
    ws = _lib.empty((need,), torch.uint8, dev) if need else None
    _lib.call_on(dev, _lib.lib().kitty_prompt_attn, "kitty_prompt_attn", q.data_ptr(), k.data_ptr(), v.data_ptr(),
                 _lib.dtype_code(q.dtype), _lib.i64_array(q_st + k_st + v_st), B, Lq, Lk, h_q, h_kv, float(scaling),
                 int(causal), *(None if x is None else x.data_ptr() for x in (q_len, k_len, cu_q, cu_k)), out.data_ptr(),
                 int(zero_rest), _status_word(dev), None if ws is None else ws.data_ptr(), need)
    if not zero_rest:
        _lib.written(out)
    return out
