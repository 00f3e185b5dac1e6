"""ctypes binding of libkitty_b200.so (declarations in include/kitty_b200.h).

There is no CPU or PyTorch fallback: if the shared library is missing or a call
fails, the error is raised to the caller.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

import torch
from torch.autograd import forward_ad

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libkitty_b200.so")

KITTY_OK, KITTY_E_BADARG, KITTY_E_BADSHAPE, KITTY_E_WORKSPACE, KITTY_E_CUDA, KITTY_E_TIMEOUT = 0, -1, -2, -3, -4, -5
KITTY_E_STATIC_LIMIT, KITTY_E_OVERLAP = -6, -7
STATIC_SCRATCH_BYTES = 8 << 20
KITTY_F16, KITTY_BF16, KITTY_F32 = 0, 1, 2
SELECT_FUSED, SELECT_SUPPLIED = 0, 1
DIV_IEEE, DIV_FULL = 0, 1
ROPE_HALF, ROPE_INTERLEAVED = 0, 1
KV8_BLOCK, KV8_RECORD, KV8_MAX_BATCH = 32, 8208, 2048
KV8_BAD_PAGE, KV8_BAD_LENGTH, KV8_TIMEOUT = 1, 2, 4

EXPORTS = [
    "kitty_version", "kitty_strerror", "kitty_quant_pack_k", "kitty_quant_pack_v", "kitty_quant_pack_kv",
    "kitty_prefill_tails",
    "kitty_append", "kitty_flush", "kitty_decode_workspace_bytes", "kitty_workspace_status", "kitty_decode_attn",
    "kitty_lse_merge", "kitty_decode_attn_static", "kitty_plan_step", "kitty_decode_step",
    "kitty_lse_exchange_bytes", "kitty_lse_exchange_merge", "kitty_decode_attn_exchange", "kitty_rope_qk",
    "kitty_plan_step_split", "kitty_decode_step_exchange", "kitty_append_rows", "kitty_flush_rows",
    "kitty_decode_attn_rows", "kitty_rotary", "kitty_prompt_workspace_bytes", "kitty_prompt_attn", "kitty_kv8_append", "kitty_kv8_expand",
    "kitty_kv8_workspace_bytes", "kitty_kv8_attn", "kitty_rows_overlap",
]


class KittyLayer(C.Structure):
    """struct kitty_layer"""
    _fields_ = [(n, C.c_int32) for n in
                ("max_bs", "max_page", "h_kv", "head_dim", "d_boost", "page_size", "sink_size", "reserved")] + \
               [(n, C.c_void_p) for n in
                ("KeyCache", "KeyCache_metadata", "ValueCache", "ValueCache_metadata", "PageTable_K", "PageTable_V",
                 "Sink_Buffer_K", "Sink_Buffer_V", "Q_Buffer_K", "Q_Buffer_V", "Local_Buffer_V")]


class KittyCounts(C.Structure):
    """struct kitty_counts"""
    _fields_ = [(n, C.c_int32) for n in
                ("PageCount_K", "PageCount_V", "Sink_Count", "Q_Buffer_Count_K", "Q_Buffer_Count_V", "Local_Count_V",
                 "Write_Offset_Local_V", "reserved")]


class KittyStepState(C.Structure):
    """struct kitty_step_state"""
    _fields_ = [("before", KittyCounts), ("after", KittyCounts), ("next", KittyCounts)] + \
               [(n, C.c_int32) for n in ("pb", "pe", "ch", "nchunk", "has_sink", "has_tail", "n_slots", "n_tiles",
                                         "chunk_slot0", "edge_slot", "n_items", "n_edge", "flush_k", "flush_v",
                                         "edge_parts", "edge_part_tok", "xchg_seq", "reserved")]


class KittyRotaryPlan(C.Structure):
    """struct kitty_rotary_plan"""
    _fields_ = [("turns", C.c_void_p), ("steps", C.c_void_p), ("factor", C.c_float), ("rotary_dim", C.c_int32), ("layout", C.c_int32),
                ("reserved", C.c_int32)]


class KittyKV8Layer(C.Structure):
    """struct kitty_kv8_layer"""
    _fields_ = [(n, C.c_int32) for n in ("max_bs", "max_page", "num_pages", "h_kv", "head_dim", "dtype")] + \
               [(n, C.c_void_p) for n in ("pages", "tail_k", "tail_v", "page_table", "status")]


_I64 = {n: struct.Struct(f"{n}q").pack for n in (3, 9, 12)}


def i64_array(values) -> bytes:
    """HOST array of int64 for the entry points that take strides that way."""
    return _I64[len(values)](*values)


class KittyError(RuntimeError):
    def __init__(self, status: int, where: str):
        self.status = status
        super().__init__(f"{where}: {strerror(status)} (status {status})")


_lib = None


def lib() -> C.CDLL:
    """The loaded library; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing. Build the CUDA library first: python -m kitty_b200.build "
            "(kitty_b200 has no CPU fallback).")
    L = C.CDLL(LIB_PATH)
    i32, i64, vp = C.c_int32, C.c_int64, C.c_void_p
    L.kitty_version.restype = C.c_int
    L.kitty_strerror.restype = C.c_char_p
    L.kitty_strerror.argtypes = [C.c_int]
    L.kitty_quant_pack_k.restype = C.c_int
    L.kitty_quant_pack_k.argtypes = [vp, C.c_int, i64, i64, i64, i32, i32, i64, i32, vp, i64, i32, vp, i64, vp, vp,
                                     C.c_int, C.c_int, vp]
    L.kitty_quant_pack_v.restype = C.c_int
    L.kitty_quant_pack_v.argtypes = [vp, C.c_int, i64, i64, i64, i32, i32, i64, i32, vp, i64, i32, vp, i64, vp,
                                     C.c_int, vp]
    L.kitty_quant_pack_kv.restype = C.c_int
    L.kitty_quant_pack_kv.argtypes = [vp, vp, C.c_int, i64, i64, i64, i64, i64, i64, i32, i32,
                                      i64, i32, vp, i64, i32, vp, i64, vp, vp, C.c_int,
                                      i64, i32, vp, i64, i32, vp, i64, vp, C.c_int, vp]
    L.kitty_prefill_tails.restype = C.c_int
    L.kitty_prefill_tails.argtypes = [C.POINTER(KittyLayer), vp, vp, C.c_int, i64, i64, i64, i64, i64, i64, i32, i64,
                                      i32, i32, i32, i32, vp]
    L.kitty_append.restype = C.c_int
    L.kitty_append.argtypes = [C.POINTER(KittyLayer), C.POINTER(KittyCounts), vp, vp, C.c_int, i64, i64, i64, i64, i32,
                               vp]
    L.kitty_flush.restype = C.c_int
    L.kitty_flush.argtypes = [C.POINTER(KittyLayer), C.POINTER(KittyCounts), i32, C.c_int, C.c_int, C.c_int, C.c_int,
                              vp]
    L.kitty_decode_workspace_bytes.restype = i64
    L.kitty_decode_workspace_bytes.argtypes = [i32, i32, i32, i32]
    L.kitty_workspace_status.restype = C.c_int
    L.kitty_workspace_status.argtypes = [vp, C.POINTER(i32), vp]
    L.kitty_decode_attn.restype = C.c_int
    L.kitty_decode_attn.argtypes = [C.POINTER(KittyLayer), C.POINTER(KittyCounts), vp, C.c_int, i32, i32, C.c_float,
                                    vp, C.c_int, vp, i64, i32, i32, i32, vp, C.c_int, vp]
    L.kitty_decode_attn_static.restype = C.c_int
    L.kitty_decode_attn_static.argtypes = [C.POINTER(KittyLayer), C.POINTER(KittyCounts), vp, C.c_int, i32, i32,
                                           C.c_float, vp, C.c_int, i32, i32, i32, vp, C.c_int, vp, vp]
    L.kitty_plan_step.restype = C.c_int
    L.kitty_plan_step.argtypes = [C.POINTER(KittyLayer), C.POINTER(KittyCounts), i32, i32, C.POINTER(KittyStepState),
                                  vp, vp]
    L.kitty_decode_step.restype = C.c_int
    L.kitty_decode_step.argtypes = [C.POINTER(KittyLayer), vp, vp, vp, C.c_int, i64, i64, i64, i64, vp, C.c_int, i32,
                                    i32, C.c_float, vp, C.c_int, vp, i64, C.c_int, vp]
    L.kitty_plan_step_split.restype = C.c_int
    L.kitty_plan_step_split.argtypes = [C.POINTER(KittyLayer), C.POINTER(KittyCounts), i32, i32, i32, i32, i32, i32,
                                        C.POINTER(KittyStepState), vp, vp]
    L.kitty_decode_step_exchange.restype = C.c_int
    L.kitty_decode_step_exchange.argtypes = [C.POINTER(KittyLayer), vp, vp, vp, C.c_int, i64, i64, i64, i64, vp, C.c_int,
                                             i32, i32, C.c_float, vp, C.c_int, vp, i64, C.c_int, vp, i32, i32, i32, vp,
                                             i64, vp]
    L.kitty_append_rows.restype = C.c_int
    L.kitty_append_rows.argtypes = [C.POINTER(KittyLayer), vp, vp, vp, vp, C.c_int, i64, i64, i64, i64, i32, vp]
    L.kitty_flush_rows.restype = C.c_int
    L.kitty_flush_rows.argtypes = [C.POINTER(KittyLayer), vp, vp, i32, C.c_int, C.c_int, vp]
    L.kitty_decode_attn_rows.restype = C.c_int
    L.kitty_decode_attn_rows.argtypes = [C.POINTER(KittyLayer), vp, vp, vp, C.c_int, i32, i32, C.c_float, vp, C.c_int,
                                         vp, i64, C.c_int, vp]
    L.kitty_decode_attn_exchange.restype = C.c_int
    L.kitty_decode_attn_exchange.argtypes = [C.POINTER(KittyLayer), C.POINTER(KittyCounts), vp, C.c_int, i32, i32,
                                             C.c_float, vp, C.c_int, vp, i64, i32, i32, i32, C.c_int, vp, i32, i32, i32,
                                             vp, i64, vp]
    L.kitty_rope_qk.restype = C.c_int
    L.kitty_rope_qk.argtypes = [vp, vp, vp, vp, vp, vp, C.c_int, i32, i32, i32, i64, vp]
    L.kitty_lse_exchange_bytes.restype = i64
    L.kitty_lse_exchange_bytes.argtypes = [i64, i32, C.POINTER(i64)]
    L.kitty_lse_exchange_merge.restype = C.c_int
    L.kitty_lse_exchange_merge.argtypes = [vp, i64, vp, i32, i32, i32, vp, C.c_int, vp, i64, vp]
    L.kitty_lse_merge.restype = C.c_int
    L.kitty_lse_merge.argtypes = [vp, i32, i64, vp, C.c_int, vp]
    rot, kv8, strides = C.POINTER(KittyRotaryPlan), C.POINTER(KittyKV8Layer), C.c_char_p
    L.kitty_rows_overlap.restype = C.c_int
    L.kitty_rows_overlap.argtypes = [vp, strides, strides, vp, strides, strides, i64]
    L.kitty_rotary.restype = C.c_int
    L.kitty_rotary.argtypes = [rot, vp, vp, vp, i64, vp, vp, C.c_int, i32, i32, i32, i32, strides, vp]
    L.kitty_prompt_attn.restype = C.c_int
    L.kitty_prompt_attn.argtypes = [vp, vp, vp, C.c_int, strides, i32, i64, i64, i32, i32, C.c_float, C.c_int, vp, vp,
                                    vp, vp, vp, C.c_int, vp, vp, i64, vp]
    L.kitty_prompt_workspace_bytes.restype = i64
    L.kitty_prompt_workspace_bytes.argtypes = [i32, i64, i64, i32, i32, C.c_int, C.c_int]
    L.kitty_kv8_append.restype = C.c_int
    L.kitty_kv8_append.argtypes = [kv8, vp, vp, strides, vp, vp, i32, i32, rot, vp, vp, i32, vp]
    L.kitty_kv8_expand.restype = C.c_int
    L.kitty_kv8_expand.argtypes = [kv8, vp, vp, vp, vp, i32, i32, vp]
    L.kitty_kv8_workspace_bytes.restype = i64
    L.kitty_kv8_workspace_bytes.argtypes = [i32, i32, i32, i32]
    L.kitty_kv8_attn.restype = C.c_int
    L.kitty_kv8_attn.argtypes = [kv8, vp, vp, i32, i32, C.c_float, vp, vp, i64, vp]
    _lib = L
    return L


def strerror(status: int) -> str:
    return lib().kitty_strerror(int(status)).decode()


def check(status: int, where: str) -> None:
    if status != KITTY_OK:
        raise KittyError(int(status), where)


_DTYPES = {torch.float16: KITTY_F16, torch.bfloat16: KITTY_BF16, torch.float32: KITTY_F32}


def dtype_code(dtype) -> int:
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise TypeError(f"kitty_b200 supports float16, bfloat16 and float32 tensors, got {dtype}") from None


def refuse_gradients(where: str, *tensors) -> None:
    """The operators are for serving: a result without a gradient, or a tangent, where one is expected would be a silent
    mistake."""
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                raise ValueError(f"{where} has no backward pass: call it under torch.no_grad() or with detached tensors")
    if forward_ad._current_level >= 0:
        for x in tensors:
            if x is not None and forward_ad.unpack_dual(x).tangent is not None:
                raise ValueError(f"{where} has no forward derivative: call it with the primal of a dual tensor")


# To be called for a lent output once it is written: a tensor that autograd has saved for a backward pass is missed there.
written = torch.autograd.graph.increment_version


def head_rows(x, repeated: bool = True):
    """x [B, H, T, 128], or [T, H, 128] for a packed batch, as the kernels read it, and its (batch, head, token) strides
    (0 where a dimension has size one: views may carry any number there).  That is x itself when its channels are
    consecutive and every row starts on a 16-byte boundary (and, without `repeated`, no dimension is expanded), otherwise
    a copy."""
    for _ in range(2):
        st, shape = x.stride(), x.shape
        if len(st) == 4:
            a, b, c, d = st
            n, m, t, _w = shape
        else:
            a, n = 0, 1
            c, b, d = st
            t, m, _w = shape
        if n < 2:
            a = 0
        if m < 2:
            b = 0
        if t < 2:
            c = 0
        if d == 1 and not (a | b | c) & (15 // x.element_size()) and not x.data_ptr() & 15 \
                and (repeated or (a or n < 2) and (b or m < 2) and (c or t < 2)):
            break
        x = x.clone(memory_format=torch.contiguous_format)
    return x, (a, b, c)


def empty(shape, dtype, device):
    """torch.empty for a contiguous tensor by the way that costs least on the host."""
    if len(shape) == 4:
        _n, h, t, d = shape
        strides = (h * t * d, t * d, d, 1)
    elif len(shape) == 3:
        strides = (shape[1] * shape[2], shape[2], 1)
    else:
        strides = (1,)
    return torch.empty_strided(shape, strides, dtype=dtype, device=device)


def call_on(device, fn, where: str, *args) -> None:
    """Call an entry point with the current stream of `device` (a CUDA device with an index) as its last argument and
    that device current, and raise if it refuses.  A small call costs more on the host than on the device, so the device
    is switched only where it has to be."""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc == KITTY_E_OVERLAP:
        raise ValueError(f"{where}: {strerror(rc)}")
    if rc != KITTY_OK:
        raise KittyError(int(rc), where)


def stream_ptr(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream
