"""Kernel bodies of the decoding ops (``csrc/kv8.cu``, ``csrc/verify.cu``); statements in :mod:`nestor_b200.ops.decode`."""

from __future__ import annotations

import ctypes as C
import math

import torch
from torch import Tensor

from nestor_b200.ops import _lib
from nestor_b200.ops import decode as D
from nestor_b200.ops.decode import BLOCK, FLOATS, KV8Cache


class CacheArgs(C.Structure):
    _fields_ = [("k_codes", C.c_void_p), ("v_codes", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("k_open", C.c_void_p), ("v_open", C.c_void_p), ("status", C.c_void_p),
                ("L", C.c_int), ("H", C.c_int), ("nb", C.c_int), ("D", C.c_int), ("U", C.c_int), ("code", C.c_int), ("type", C.c_int)]


class RowArgs(C.Structure):      # (pairs of the C structure, keys then values, are two fields here: cheaper to fill)
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_row", C.c_long), ("v_row", C.c_long), ("k_head", C.c_long),
                ("v_head", C.c_long), ("k_out", C.c_void_p), ("v_out", C.c_void_p), ("seg", C.c_void_p), ("start", C.c_void_p), ("rows", C.c_int), ("max_rows", C.c_int)]


class AttentionArgs(C.Structure):
    _fields_ = [("q", C.c_void_p), ("out", C.c_void_p), ("q_row", C.c_long), ("q_head", C.c_long), ("o_row", C.c_long), ("o_head", C.c_long),
                ("seg", C.c_void_p), ("len", C.c_void_p), ("rows", C.c_int), ("max_rows", C.c_int), ("group", C.c_int), ("q_type", C.c_int),
                ("zero_tail", C.c_int), ("scale_log2", C.c_float)]


class VerifyArgs(C.Structure):
    _fields_ = [("p", C.c_void_p), ("q", C.c_void_p), ("tokens", C.c_void_p), ("u", C.c_void_p), ("w", C.c_void_p), ("len", C.c_void_p),
                ("accepted", C.c_void_p), ("token", C.c_void_p), ("p_batch", C.c_long), ("p_row", C.c_long), ("q_batch", C.c_long),
                ("q_row", C.c_long), ("B", C.c_int), ("n", C.c_int), ("V", C.c_int), ("type", C.c_int), ("tokens_64", C.c_int)]


_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_ready = None


def _L():
    global _ready
    if _ready is None:
        L = _lib.lib()
        vp, p = C.c_void_p, C.POINTER
        L.nb_kv8_append.argtypes = [p(CacheArgs), p(RowArgs), vp]
        L.nb_kv8_truncate.argtypes = [p(CacheArgs), vp, vp]
        L.nb_kv8_read.argtypes = [p(CacheArgs), p(RowArgs), C.c_int, vp]
        L.nb_kv8_attention.argtypes = [p(CacheArgs), p(AttentionArgs), vp, C.c_long, C.c_uint, vp]
        L.nb_kv8_attention_workspace.argtypes = [C.c_int] * 7
        L.nb_verify_draft.argtypes = [p(VerifyArgs), vp]
        for f in (L.nb_kv8_append, L.nb_kv8_truncate, L.nb_kv8_read, L.nb_kv8_attention, L.nb_verify_draft):
            f.restype = C.c_int
        L.nb_kv8_attention_workspace.restype = C.c_long
        _ready = L
    return _ready


def _launch(fn, device: torch.device, *args, launches: int = 1) -> None:
    """Call an entry point with the current stream of ``device`` (which need not be the current device)."""

    # (the raw-stream query costs a tenth of torch.cuda.current_stream(), which builds a Stream object)
    index = device.index
    if _device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        raise RuntimeError(f"{fn.__name__} failed with code {rc}")
    _lib.count_launch(launches)


def _cache_args(c: KV8Cache) -> CacheArgs:
    a = c.__dict__.get("_args")          # (the fields are fixed: one argument block serves every call)
    if a is None:
        a = CacheArgs(c.k_codes.data_ptr(), c.v_codes.data_ptr(), c.k_scale.data_ptr(), c.v_scale.data_ptr(), c.k_open.data_ptr(),
                      c.v_open.data_ptr(), _lib.status_word(c.device).data_ptr(), c.lists, c.heads, c.blocks, c.head_dim, c.units,
                      0 if c.dtype == torch.int8 else 1, FLOATS[c.open_dtype])
        c.__dict__["_args"] = a
    return a


def _rows(t: Tensor) -> Tensor:
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def kv8_append(cache: KV8Cache, k: Tensor, v: Tensor, seg_start: Tensor, start: Tensor, max_rows: int = 1) -> None:
    D.check_append(cache, k, v, seg_start, start, max_rows)
    if k.shape[0] == 0:
        return
    k, v = _rows(k), _rows(v)
    (k_row, k_head, _), (v_row, v_head, _) = k.stride(), v.stride()
    a = RowArgs(k.data_ptr(), v.data_ptr(), k_row, v_row, k_head, v_head, None, None, seg_start.data_ptr(), start.data_ptr(),
                k.shape[0], min(max_rows, k.shape[0]))
    _launch(_L().nb_kv8_append, cache.device, _cache_args(cache), a)


def kv8_truncate(cache: KV8Cache, lengths: Tensor) -> None:
    D.check_index(lengths, cache.lists, "lengths", cache.device)
    _launch(_L().nb_kv8_truncate, cache.device, _cache_args(cache), lengths.data_ptr())


def kv8_read(cache: KV8Cache, seg_start: Tensor, start: Tensor, rows: int, dtype: torch.dtype = torch.float32,
             max_rows: int = BLOCK) -> tuple[Tensor, Tensor]:
    D.check_read(cache, seg_start, start, rows, dtype, max_rows)
    k = torch.empty(rows, cache.heads, cache.head_dim, dtype=dtype, device=cache.device)
    v = torch.empty_like(k)
    if rows:
        a = RowArgs(None, None, 0, 0, 0, 0, k.data_ptr(), v.data_ptr(), seg_start.data_ptr(), start.data_ptr(), rows, min(max_rows, 1 << 30))
        _launch(_L().nb_kv8_read, cache.device, _cache_args(cache), a, FLOATS[dtype])
    return k, v


LOG2E = math.log2(math.e)
WAIT_POLLS = 1 << 24       # looks at a copy of codes before the attention's wait for it gives up (status word, NaN rows)
_sizes: dict = {}          # bytes of workspace for a shape (a function of the shape and the device alone)


def kv8_attention(q: Tensor, cache: KV8Cache, seg_start: Tensor, lengths: Tensor, scale: float, max_rows: int = 1,
                  out: Tensor | None = None) -> Tensor:
    D.check_attention(q, cache, seg_start, lengths, scale, max_rows, out)
    given = out is not None
    if not given:
        out = q.new_empty(q.shape)
    rows = q.shape[0]
    if rows == 0:
        return out
    q = _rows(q)
    q_row, q_head, _ = q.stride()
    o_row, o_head, _ = out.stride()
    group, max_rows = q.shape[1] // cache.heads, min(max_rows, rows)
    L = _L()
    key = (cache.lists, cache.heads, cache.blocks, cache.head_dim, rows, max_rows, group)
    size = _sizes.get((cache.device.index, key))
    if size is None:
        with torch.cuda.device(cache.device):
            size = L.nb_kv8_attention_workspace(*key)
        if len(_sizes) >= 4096:
            _sizes.clear()
        _sizes[cache.device.index, key] = size
    # (allocated for this call on this stream: two streams, or two captured graphs, never share it)
    ws = lengths.new_empty(-(-size // 4)) if size else None
    a = AttentionArgs(q.data_ptr(), out.data_ptr(), q_row, q_head, o_row, o_head, seg_start.data_ptr(), lengths.data_ptr(), rows,
                      max_rows, group, FLOATS[q.dtype], 0 if given else 1, scale * LOG2E)
    _launch(L.nb_kv8_attention, cache.device, _cache_args(cache), a, None if ws is None else ws.data_ptr(), size, WAIT_POLLS,
            launches=1 if ws is None else 2)
    return out


def verify_draft(target_probs: Tensor, draft_tokens: Tensor, draft_probs: Tensor | None, accept_u: Tensor, sample_u: Tensor,
                 draft_len: Tensor | None = None) -> tuple[Tensor, Tensor]:
    D.check_verify(target_probs, draft_tokens, draft_probs, accept_u, sample_u, draft_len)
    p, q = target_probs, draft_probs
    B, n, V = p.shape
    n -= 1
    out = torch.empty(2, B, dtype=torch.int32, device=p.device)
    accepted, token = out.unbind(0)
    if B == 0:
        return accepted, token
    if V > 1 and p.stride(2) != 1:
        p = p.contiguous()
    if n == 0:
        q = None
    elif q is not None and V > 1 and q.stride(2) != 1:
        q = q.contiguous()
    p_batch, p_row, _ = p.stride()
    q_batch, q_row, _ = (0, 0, 0) if q is None else q.stride()
    draft_tokens, accept_u, sample_u = draft_tokens.contiguous(), accept_u.contiguous(), sample_u.contiguous()
    at = out.data_ptr()
    a = VerifyArgs(p.data_ptr(), None if q is None else q.data_ptr(), draft_tokens.data_ptr(), accept_u.data_ptr(), sample_u.data_ptr(),
                   None if draft_len is None else draft_len.data_ptr(), at, at + 4 * B, p_batch, p_row, q_batch, q_row, B, n, V,
                   FLOATS[p.dtype], 1 if draft_tokens.dtype == torch.int64 else 0)
    _launch(_L().nb_verify_draft, p.device, a)
    return accepted, token
