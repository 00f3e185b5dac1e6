"""The 8-bit cache: pages of 128 tokens behind a page table, a scale for each block of 32 tokens and head.

For layers or models that two bits per value hurt: keys and values are whole numbers -127..127 times one fp32 scale per
(block, head), off by at most 1/254 (0.39 %) of the block's largest and half the size of a 16-bit cache.  The tokens of a
row's open block stay in 16 bits until it is full, as `KittyCache` keeps its Q-buffers, so what is stored does not depend
on how the tokens were cut into calls.

The caller keeps the lengths and passes them as device tensors (`start`, `lengths`: int32, one per row), so every call
can be captured in a CUDA graph and replayed as the sequences grow; `KV8Layer.check()` reports what the kernels had to
skip or clamp.  The reference has no such cache.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from .rotary import RotaryEmbedding

PAGE_SIZE = 128
BLOCK = _lib.KV8_BLOCK
_TYPES = (torch.float16, torch.bfloat16)


class KV8Layer:
    """Device buffers of one layer's 8-bit cache.

    MAX_BS rows of up to MAX_LEN tokens, H_KV heads of 128 channels; dtype (fp16 or bf16) is the type of the open blocks,
    of the tokens that come in and of the values that go out.  page_table: int64 [MAX_BS, ceil(MAX_LEN / 128)] page rows
    (default: row b's pages side by side); num_pages: page rows of the cache (default: as many as the table has
    entries).  The table, `layer.page_table`, may be changed between calls, in place or for another contiguous one (one that
    is not contiguous is copied when the layer is made); entries of pages that no token has reached are never read."""

    def __init__(self, MAX_BS: int, MAX_LEN: int, H_KV: int, D: int = 128, *, dtype: torch.dtype = torch.bfloat16,
                 device="cuda", num_pages: Optional[int] = None, page_table: Optional[torch.Tensor] = None):
        if D != 128:
            raise ValueError(f"kitty_b200 kernels are built for D=128, got {D}")
        if MAX_BS <= 0 or MAX_LEN <= 0 or H_KV <= 0:
            raise ValueError(f"MAX_BS, MAX_LEN and H_KV must be positive, got {(MAX_BS, MAX_LEN, H_KV)}")
        if MAX_LEN > 1 << 30:
            raise ValueError(f"MAX_LEN is limited to 2^30 tokens, got {MAX_LEN}")
        if dtype not in _TYPES:
            raise TypeError(f"the 8-bit cache takes float16 or bfloat16 tokens, got {dtype}")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("kitty_b200 buffers live on a CUDA device (there is no CPU path)")
        self.MAX_BS, self.MAX_LEN, self.H_KV, self.D, self.dtype = MAX_BS, MAX_LEN, H_KV, D, dtype
        self.MAX_PAGE = math.ceil(MAX_LEN / PAGE_SIZE)
        n = MAX_BS * self.MAX_PAGE if num_pages is None else int(num_pages)
        if n <= 0:
            raise ValueError(f"num_pages must be positive, got {num_pages}")
        if page_table is None:
            if num_pages is not None and n < MAX_BS * self.MAX_PAGE:
                raise ValueError("a cache with fewer page rows than its table has entries needs a page_table")
            page_table = torch.arange(MAX_BS * self.MAX_PAGE, dtype=torch.int64, device=dev).view(MAX_BS, self.MAX_PAGE)
        if tuple(page_table.shape) != (MAX_BS, self.MAX_PAGE) or page_table.dtype != torch.int64:
            raise ValueError(f"page_table must be int64 [{MAX_BS}, {self.MAX_PAGE}], got "
                             f"{page_table.dtype} {tuple(page_table.shape)}")
        self.num_pages = n
        self.pages = torch.zeros((n, H_KV, PAGE_SIZE // BLOCK, _lib.KV8_RECORD), dtype=torch.uint8, device=dev)
        self.device = self.pages.device
        if page_table.device != self.device:
            raise ValueError(f"page_table is on {page_table.device}, the cache on {self.device}")
        self.page_table = page_table.contiguous()
        self.tail_k = torch.zeros((MAX_BS, H_KV, BLOCK, D), dtype=dtype, device=dev)
        self.tail_v = torch.zeros((MAX_BS, H_KV, BLOCK, D), dtype=dtype, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._workspace_need: dict = {}
        self._c_layer = self._c_table = None

    def c_layer(self) -> "_lib.KittyKV8Layer":
        """struct kitty_kv8_layer.  The buffers are the constructor's; the page table may have been replaced."""
        L = self._c_layer
        table = self.page_table
        if L is None:
            L = _lib.KittyKV8Layer(self.MAX_BS, self.MAX_PAGE, self.num_pages, self.H_KV, self.D,
                                   _lib.dtype_code(self.dtype))
            for name in ("pages", "tail_k", "tail_v", "status"):
                t = getattr(self, name)
                assert t.is_contiguous() and t.device == self.device, name
                setattr(L, name, t.data_ptr())
            self._c_layer = L
        if self._c_table is not table:
            if tuple(table.shape) != (self.MAX_BS, self.MAX_PAGE) or table.dtype != torch.int64 \
                    or table.device != self.device or not table.is_contiguous():
                raise ValueError(f"page_table must be contiguous int64 [{self.MAX_BS}, {self.MAX_PAGE}] on {self.device}")
            # a new struct: another thread's call may be reading the old one
            L = self._c_layer = _lib.KittyKV8Layer.from_buffer_copy(L)
            L.page_table = table.data_ptr()
            self._c_table = table
        return L

    def check(self) -> None:
        """Synchronise and raise if a kernel met a bad page-table entry, a bad length, or a wait that ran out."""
        st = int(self.status.item())
        if st & _lib.KV8_TIMEOUT:
            raise _lib.KittyError(_lib.KITTY_E_TIMEOUT, "KV8Layer")
        if st:
            what = [text for bit, text in ((_lib.KV8_BAD_PAGE, "a page-table entry out of range (its block was skipped)"),
                                           (_lib.KV8_BAD_LENGTH, "a length or start outside the cache (it was clamped)"))
                    if st & bit]
            raise ValueError("the 8-bit cache met " + " and ".join(what))

    def workspace_bytes(self, batch: int, h_q: int) -> int:
        need = self._workspace_need.get((batch, h_q))
        if need is None:
            with torch.cuda.device(self.device):        # the plan depends on the device's multiprocessors
                need = int(_lib.lib().kitty_kv8_workspace_bytes(batch, self.H_KV, h_q, self.MAX_PAGE))
            if need < 0:
                _lib.check(need, "kitty_kv8_workspace_bytes")
            self._workspace_need[(batch, h_q)] = need
        return need


def _row_tensor(x: torch.Tensor, what: str, B: int, layer: KV8Layer) -> torch.Tensor:
    if not isinstance(x, torch.Tensor) or x.dtype != torch.int32 or x.shape != (B,) or x.device != layer.device:
        raise ValueError(f"{what} must be an int32 tensor [{B}] on {layer.device}")
    return x if x.is_contiguous() else x.contiguous()


def _tokens(x: torch.Tensor, what: str, heads: int, layer: KV8Layer):
    shape = x.shape
    if len(shape) != 4 or shape[1] != heads or shape[3] != layer.D:
        raise ValueError(f"expected {what} [B, {heads}, T, {layer.D}], got {tuple(shape)}")
    if x.dtype != layer.dtype or x.device != layer.device:
        if not x.is_cuda:
            raise ValueError(f"kitty_b200 has no CPU path: the {what} must be on a CUDA device")
        raise ValueError(f"the {what} must be {layer.dtype} on {layer.device}, got {x.dtype} on {x.device}")
    return _lib.head_rows(x)


def kv8_append(layer: KV8Layer, key: torch.Tensor, value: torch.Tensor, start: torch.Tensor, *,
               lengths: Optional[torch.Tensor] = None, rotary: Optional[RotaryEmbedding] = None,
               query: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Append tokens key / value [B, H, T, 128] (any strides with consecutive channels) to rows 0 .. B-1.

    start: int32 [B], the tokens each row holds already (a row may be cut back to any length within its open block;
    further back, give the tokens again from that block's first one).  lengths: int32 [B], how many of the T tokens are the row's
    (default all).  rotary: the keys are turned on the way, token i of row b by position start[b] + i.  query
    [B, H_Q, T, 128] is then turned by the same positions and returned, [B, H_Q, T, 128] contiguous (all T tokens);
    without it the call returns None."""
    _lib.refuse_gradients("kv8_append", key, value, query)
    (k, k_st), (v, v_st) = _tokens(key, "key", layer.H_KV, layer), _tokens(value, "value", layer.H_KV, layer)
    B, _, T, _ = k.shape
    if v.shape != k.shape:
        raise ValueError(f"key and value differ in shape: {tuple(k.shape)} and {tuple(v.shape)}")
    if B > layer.MAX_BS:
        raise ValueError(f"{B} rows in a cache of {layer.MAX_BS}")
    if T > layer.MAX_PAGE * PAGE_SIZE:
        raise _lib.KittyError(_lib.KITTY_E_BADARG, "kv8_append: the tokens do not fit the cache's pages")
    start = _row_tensor(start, "start", B, layer)
    if lengths is not None:
        lengths = _row_tensor(lengths, "lengths", B, layer)
    out, h_q, q_st = None, 0, (0, 0, 0)
    if query is not None:
        if rotary is None:
            raise ValueError("the query goes along to be turned: pass rotary")
        if query.dim() != 4 or query.shape[0] != B or query.shape[2] != T:
            raise ValueError(f"expected query [{B}, H_Q, {T}, {layer.D}], got {tuple(query.shape)}")
        h_q = query.shape[1]
        query, q_st = _tokens(query, "query", h_q, layer)
        out = _lib.empty((B, h_q, T, layer.D), layer.dtype, layer.device)
    if rotary is not None and rotary.device != layer.device:
        raise ValueError(f"the angles are on {rotary.device}, the cache on {layer.device}")
    _lib.call_on(layer.device, _lib.lib().kitty_kv8_append, "kitty_kv8_append", layer.c_layer(), k.data_ptr(),
                 v.data_ptr(), _lib.i64_array(k_st + v_st + q_st), start.data_ptr(), None if lengths is None else lengths.data_ptr(),
                 B, T, None if rotary is None else rotary.c_plan(), query.data_ptr() if h_q else None,
                 out.data_ptr() if h_q else None, h_q)
    return out


def kv8_expand(layer: KV8Layer, lengths: torch.Tensor, n: int, *, start: Optional[torch.Tensor] = None):
    """Tokens start[b] .. start[b] + n - 1 (default from 0) of rows that hold lengths[b] tokens, as 16-bit values:
    (key, value) [B, H, n, 128] of the layer's type, zeros behind a row's last token.  What a further piece of a prompt
    attends to (`prompt_attention` with more keys than queries)."""
    if not isinstance(lengths, torch.Tensor) or lengths.dim() != 1:
        raise ValueError("lengths must be an int32 tensor [B]")
    B, n = lengths.shape[0], int(n)
    if B > layer.MAX_BS or n < 0 or n > 1 << 30:
        raise ValueError(f"{B} rows of {n} tokens from a cache of {layer.MAX_BS} rows")
    lengths = _row_tensor(lengths, "lengths", B, layer)
    if start is not None:
        start = _row_tensor(start, "start", B, layer)
    shape = (B, layer.H_KV, n, layer.D)
    k, v = _lib.empty(shape, layer.dtype, layer.device), _lib.empty(shape, layer.dtype, layer.device)
    _lib.call_on(layer.device, _lib.lib().kitty_kv8_expand, "kitty_kv8_expand", layer.c_layer(), lengths.data_ptr(),
                 None if start is None else start.data_ptr(), k.data_ptr(), v.data_ptr(), B, n)
    return k, v


def kv8_attention(query: torch.Tensor, layer: KV8Layer, lengths: torch.Tensor, scaling: float, *,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one query token per row over the lengths[b] tokens (int32 [B], on the device) that row b holds.
    query [B, H_Q, 1, 128] of the layer's type, up to 16 query heads per key head.  Returns [B, 1, H_Q, 128]; a row
    without tokens is zero.  `out` may be a view of the query's own memory, row for row; other overlaps are refused.  The
    scratch is the caller's stream's (torch's allocator), so calls may run side by side."""
    if query.dim() != 4 or query.shape[2] != 1:
        raise ValueError(f"expected query [B, H_Q, 1, {layer.D}], got {tuple(query.shape)}")
    _lib.refuse_gradients("kv8_attention", query, out)
    B, h_q, _, D = query.shape
    q, _ = _tokens(query, "query", h_q, layer)
    if h_q == 0 or h_q % layer.H_KV:
        raise ValueError(f"{h_q} query heads over {layer.H_KV} key heads")
    if B > layer.MAX_BS:
        raise ValueError(f"{B} rows in a cache of {layer.MAX_BS}")
    q = q.contiguous()
    lengths = _row_tensor(lengths, "lengths", B, layer)
    need = layer.workspace_bytes(B, h_q)
    lent = out is not None
    if out is None:
        out = _lib.empty((B, 1, h_q, D), layer.dtype, layer.device)
    elif tuple(out.shape) != (B, 1, h_q, D) or out.dtype != layer.dtype or out.device != layer.device \
            or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {layer.dtype} [{B}, 1, {h_q}, {D}] on {layer.device}")
    ws = _lib.empty((need,), torch.uint8, layer.device) if need else None
    _lib.call_on(layer.device, _lib.lib().kitty_kv8_attn, "kitty_kv8_attn", layer.c_layer(), lengths.data_ptr(),
                 q.data_ptr(), B, h_q, float(scaling), out.data_ptr(), None if ws is None else ws.data_ptr(), need)
    if lent:
        _lib.written(out)
    return out
