"""Decoding with an 8-bit key/value cache: the cache, argument checks, and the PyTorch statement of every op.

A *list* is what one attention column has seen of one sequence (``list = column * B + sequence``, the order of
``ColumnPlan``). The rows of a step are packed by list: list ``l`` owns rows ``seg_start[l] : seg_start[l + 1]``.

The cache of a (list, head) is a run of blocks of 64 entries. The keys and the values of a block each have one fp32
scale; a value is ``code * scale``. With ``Q = 127`` (int8) or ``448`` (e4m3) and ``amax`` the largest magnitude in the
block, ``scale = amax / Q`` and ``code = round_half_even(x * (Q / amax))`` (factor and product rounded to fp32).
A block below ``2^-100`` holds zeros; a block with an infinity or a NaN has the scale NaN. The originals of the youngest
two blocks of every list are kept, so a block that is still filling is always quantised from originals: its codes are a
function of its contents, not of the order in which they came. A list can step back to any length that is at most 64
entries below the greatest it has had, and to any multiple of 64.

Kernel bodies: :mod:`nestor_b200.ops.cuda_decode`. None of these ops has a backward pass.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor
from torch.autograd import forward_ad

BLOCK = 64                                                     # entries of a block
MAX_HEAD_DIM = 128
CODE_MAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FLOATS = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class KV8Cache:
    """Keys and values of ``L`` lists in 8 bits (build an empty one with :func:`kv8_cache`).

    Attributes (fixed once built):
        k_codes, v_codes: ``[L, H, blocks, ceil(head_dim / 8), 512]`` int8 or float8_e4m3fn. A block's codes are units of
            8 head dims x 64 entries in the order of the kernels' matrix fragments (:func:`code_positions`); codes of dims
            past ``head_dim`` are zero.
        k_scale, v_scale: ``[L, H, blocks]`` fp32.
        k_open, v_open: ``[L, H, 2, 64, head_dim]`` originals of the youngest two blocks (block ``b`` in slot ``b % 2``),
            in the dtype of the rows that are appended (bf16, fp16 or fp32).
        lists, heads, blocks, units, capacity, head_dim, device, is_cuda, dtype, open_dtype: what the tensors say.

    How many entries each list holds is not part of the cache: the caller keeps ``lengths [L]`` (int32, on the device)
    and passes it, so stepping back is a smaller number plus :func:`kv8_truncate`.
    """

    def __init__(self, k_codes: Tensor, v_codes: Tensor, k_scale: Tensor, v_scale: Tensor, k_open: Tensor, v_open: Tensor) -> None:
        code, kind = k_codes.dtype, k_open.dtype
        if code not in CODE_MAX or v_codes.dtype != code:
            raise ValueError(f"cache codes are int8 or float8_e4m3fn (keys and values alike), got {code} and {v_codes.dtype}")
        if kind not in FLOATS or v_open.dtype != kind:
            raise ValueError(f"the kept originals are bfloat16, float16 or float32 (keys and values alike), got {kind} and {v_open.dtype}")
        if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise ValueError("cache scales are float32")
        shape, held = k_codes.shape, k_open.shape
        if len(shape) != 5 or len(held) != 5:
            raise ValueError("cache codes are [L, H, blocks, units, 512], originals [L, H, 2, 64, head_dim]")
        L, H, nb, U, _ = shape
        D = held[4]
        if L < 1 or H < 1 or nb < 1 or not 1 <= D <= MAX_HEAD_DIM or U != -(-D // 8):
            raise ValueError(f"cache of {L} lists x {H} heads x {nb} blocks x {U} units for head_dim {D}: needs at least one of "
                             f"each, head_dim in 1..{MAX_HEAD_DIM} and ceil(head_dim / 8) units")
        device = k_codes.device
        scales = (L, H, nb)
        if not (shape == (L, H, nb, U, 512) == v_codes.shape and k_scale.shape == scales == v_scale.shape
                and held == (L, H, 2, BLOCK, D) == v_open.shape):
            raise ValueError(f"cache tensors of unlike shapes: codes {tuple(shape)} and {tuple(v_codes.shape)}, scales {tuple(k_scale.shape)} and "
                             f"{tuple(v_scale.shape)}, originals {tuple(held)} and {tuple(v_open.shape)}")
        tensors = (k_codes, v_codes, k_scale, v_scale, k_open, v_open)
        for t in tensors:
            if t.device != device or not t.is_contiguous():
                raise ValueError(f"cache tensors must be contiguous and on one device, {device}; got {tuple(t.shape)} with strides {t.stride()} on {t.device}")
        if k_codes.data_ptr() % 16 or v_codes.data_ptr() % 16:
            raise ValueError("cache codes must begin on a 16-byte boundary")
        if nb * BLOCK >= 2 ** 31:
            raise ValueError(f"a list holds fewer than 2^31 entries, got {nb} blocks")
        self.__dict__.update(k_codes=k_codes, v_codes=v_codes, k_scale=k_scale, v_scale=v_scale, k_open=k_open, v_open=v_open,
                             lists=L, heads=H, blocks=nb, units=U, capacity=nb * BLOCK, head_dim=D, device=device,
                             is_cuda=device.type == "cuda", dtype=code, open_dtype=kind)
        if self.is_cuda:
            from nestor_b200.ops import _lib
            _lib.status_word(device)             # (made here, not by a first step that may be under graph capture)

    def __setattr__(self, name: str, value) -> None:
        raise AttributeError(f"the {name} of a KV8Cache is fixed (its kernels keep an argument block of it); build another one")

    def __reduce__(self):
        # (copies and pickles are built from the tensors, so they say where their own tensors are)
        return KV8Cache, (self.k_codes, self.v_codes, self.k_scale, self.v_scale, self.k_open, self.v_open)


def kv8_cache(lists: int, heads: int, capacity: int, head_dim: int, device=None, dtype: torch.dtype = torch.int8,
              open_dtype: torch.dtype = torch.bfloat16) -> KV8Cache:
    """An empty cache: ``lists`` lists of up to ``capacity`` entries (rounded up to whole blocks)."""

    if dtype not in CODE_MAX:
        raise ValueError(f"cache codes are int8 or float8_e4m3fn, got {dtype}")
    if not 1 <= head_dim <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be in 1..{MAX_HEAD_DIM}, got {head_dim}")
    nb = max(1, -(-capacity // BLOCK))
    codes = lambda: torch.zeros(lists, heads, nb, -(-head_dim // 8), 512, dtype=torch.uint8, device=device).view(dtype)   # noqa: E731
    scale = lambda: torch.zeros(lists, heads, nb, dtype=torch.float32, device=device)                       # noqa: E731
    held = lambda: torch.zeros(lists, heads, 2, BLOCK, head_dim, dtype=open_dtype, device=device)           # noqa: E731
    return KV8Cache(codes(), codes(), scale(), scale(), held(), held())


# ----------------------------------------------------------------------------- argument checks (both bodies)
def check_index(t: Tensor, n: int, name: str, device: torch.device) -> None:
    if t.dtype != torch.int32 or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} entries on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def check_no_grad(op: str, *tensors: Tensor | None) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{op} is a decoding op without a backward pass: call it under torch.no_grad()")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{op} is a decoding op without derivatives: it takes no dual tensors")


def check_count(op: str, rows: int, max_rows: int) -> None:
    if max_rows < 1:
        raise ValueError(f"{op}: max_rows must be at least 1, got {max_rows}")
    if not 0 <= rows < 2 ** 31:
        raise ValueError(f"{op}: rows must be in 0..2^31 - 1, got {rows}")


def check_rows(op: str, t: Tensor, name: str, cache: KV8Cache) -> None:
    shape = t.shape
    if len(shape) != 3 or shape[1] != cache.heads or shape[2] != cache.head_dim or t.dtype != cache.open_dtype or t.device != cache.device:
        raise ValueError(f"{op}: {name} must be [rows, {cache.heads}, {cache.head_dim}] {cache.open_dtype} on {cache.device}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")


def check_append(cache: KV8Cache, k: Tensor, v: Tensor, seg_start: Tensor, start: Tensor, max_rows: int) -> None:
    check_no_grad("kv8_append", k, v)
    check_rows("kv8_append", k, "k", cache)
    check_rows("kv8_append", v, "v", cache)
    if v.shape[0] != k.shape[0]:
        raise ValueError(f"kv8_append: {k.shape[0]} rows of keys but {v.shape[0]} of values")
    check_index(seg_start, cache.lists + 1, "seg_start", cache.device)
    check_index(start, cache.lists, "start", cache.device)
    check_count("kv8_append", k.shape[0], max_rows)


def check_read(cache: KV8Cache, seg_start: Tensor, start: Tensor, rows: int, dtype: torch.dtype, max_rows: int) -> None:
    check_index(seg_start, cache.lists + 1, "seg_start", cache.device)
    check_index(start, cache.lists, "start", cache.device)
    check_count("kv8_read", rows, max_rows)
    if dtype not in FLOATS:
        raise ValueError(f"kv8_read writes bfloat16, float16 or float32, got {dtype}")


def check_attention(q: Tensor, cache: KV8Cache, seg_start: Tensor, lengths: Tensor, scale: float, max_rows: int, out: Tensor | None) -> None:
    check_no_grad("kv8_attention", q, out)
    shape = q.shape
    if (len(shape) != 3 or shape[2] != cache.head_dim or shape[1] < 1 or shape[1] % cache.heads or q.dtype not in FLOATS
            or q.device != cache.device):
        raise ValueError(f"kv8_attention: q must be [rows, a multiple of {cache.heads}, {cache.head_dim}] bfloat16, float16 or float32 on "
                         f"{cache.device}, got {tuple(q.shape)} {q.dtype} on {q.device}")
    check_index(seg_start, cache.lists + 1, "seg_start", cache.device)
    check_index(lengths, cache.lists, "lengths", cache.device)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"kv8_attention: scale must be positive and finite, got {scale}")
    check_count("kv8_attention", shape[0], max_rows)
    columns = shape[0] * (shape[1] // cache.heads)
    if columns > 2 ** 30 or cache.heads * -(-columns // 8) * cache.blocks >= 2 ** 31:
        raise ValueError(f"kv8_attention: {shape[0]} rows x {shape[1]} heads over {cache.blocks} blocks are too many for one call: pass them in parts")
    if out is not None:
        step = out.stride()
        if (out.shape != shape or out.dtype != q.dtype or out.device != q.device or (shape[2] > 1 and step[2] != 1)
                or (shape[0] > 1 and step[0] == 0) or (shape[1] > 1 and step[1] == 0)):
            raise ValueError(f"kv8_attention: out must have the shape, dtype and device of q, contiguous heads and rows of its own, got "
                             f"{tuple(out.shape)} {out.dtype} on {out.device}, strides {step}")


def check_verify(p: Tensor, tokens: Tensor, q: Tensor | None, u: Tensor, w: Tensor, draft_len: Tensor | None) -> None:
    check_no_grad("verify_draft", p, q)
    shape, kind, device = p.shape, p.dtype, p.device
    if len(shape) != 3 or shape[1] < 1 or shape[2] < 1 or kind not in FLOATS:
        raise ValueError(f"verify_draft: target_probs must be [B, n + 1, V] bfloat16, float16 or float32, got {tuple(shape)} {kind}")
    B, n, V = shape
    drafted = (B, n - 1)
    if tokens.shape != drafted or tokens.dtype not in (torch.int32, torch.int64) or tokens.device != device:
        raise ValueError(f"verify_draft: draft_tokens must be {drafted} int32 or int64 on {device}, got {tuple(tokens.shape)} {tokens.dtype} on {tokens.device}")
    if q is not None and (q.shape != (B, n - 1, V) or q.dtype != kind or q.device != device):
        raise ValueError(f"verify_draft: draft_probs must be {(B, n - 1, V)} {kind} on {device}, got {tuple(q.shape)} {q.dtype} on {q.device}")
    if u.shape != drafted or u.dtype != torch.float32 or u.device != device:
        raise ValueError(f"verify_draft: accept_u must be {drafted} float32 on {device}, got {tuple(u.shape)} {u.dtype} on {u.device}")
    if w.shape != (B,) or w.dtype != torch.float32 or w.device != device:
        raise ValueError(f"verify_draft: sample_u must be {(B,)} float32 on {device}, got {tuple(w.shape)} {w.dtype} on {w.device}")
    if draft_len is not None:
        check_index(draft_len, B, "draft_len", device)


# -------------------------------------------------------------------------------------- statements: the cache
_positions: dict = {}


def code_positions(which: str, units: int, device: torch.device) -> Tensor:
    """Index of entry ``e``, dim ``d`` among the ``units * 512`` codes of a block: ``[64, 8 * units]``. A unit holds 8 dims
    as 32 lanes ``(g, t)`` of 16 codes ``(m, h, i)``: keys ``e = 16m + 8h + g, d = 2t + i``; values
    ``e = 16m + 8h + 2t + i, d = g``."""

    key = (which, units, device)
    if key not in _positions:
        e = torch.arange(BLOCK, device=device).unsqueeze(1)
        d = torch.arange(8 * units, device=device).unsqueeze(0)
        r = d % 8
        lane = 4 * (e % 8) + r // 2 if which == "k" else 4 * r + (e % 8) // 2
        i = d % 2 if which == "k" else e % 2
        _positions[key] = (d // 8) * 512 + lane * 16 + (e // 16) * 4 + (e % 16) // 8 * 2 + i
    return _positions[key]


def _store_block(cache: KV8Cache, which: str, l: int, b: int, x: Tensor) -> None:
    """Quantise ``x [n <= 64, H, D]`` as the contents of block ``b`` of list ``l``."""

    codes, scale = (cache.k_codes, cache.k_scale) if which == "k" else (cache.v_codes, cache.v_scale)
    x = x.float()
    top = CODE_MAX[codes.dtype]
    amax = x.abs().amax(dim=(0, 2))                                              # (a NaN stays)
    poison = ~torch.isfinite(amax)
    empty = amax < 2.0 ** -100
    amax = torch.where(empty, 0.0, amax)
    fit = torch.where(empty | poison, 0.0, torch.full_like(amax, top) / amax)
    y = torch.where(fit[None, :, None] == 0, 0.0, x * fit[None, :, None]).clamp(-top, top)
    y = y.round().to(torch.int8) if codes.dtype == torch.int8 else y.to(codes.dtype)
    H, D = y.shape[1], y.shape[2]
    flat = torch.zeros(H, codes.shape[3] * 512, dtype=torch.uint8, device=y.device)
    at = code_positions(which, codes.shape[3], y.device)[: y.shape[0], :D]
    flat[:, at] = y.view(torch.uint8).transpose(0, 1)
    codes[l, :, b] = flat.view(codes.dtype).view(H, codes.shape[3], 512)
    scale[l, :, b] = torch.where(poison, math.nan, amax / torch.full_like(amax, top))


def _load_entries(cache: KV8Cache, which: str, l: int, first: int, n: int) -> Tensor:
    """Entries ``first : first + n`` of list ``l`` as fp32 ``[n, H, D]``."""

    codes, scale = (cache.k_codes, cache.k_scale) if which == "k" else (cache.v_codes, cache.v_scale)
    H, U = codes.shape[1], codes.shape[3]
    if n == 0:
        return torch.zeros(0, H, cache.head_dim, device=codes.device)
    b0, b1 = first // BLOCK, (first + n - 1) // BLOCK + 1
    at = code_positions(which, U, codes.device)[:, : cache.head_dim]
    raw = codes[l, :, b0:b1].reshape(H, b1 - b0, U * 512).view(torch.uint8)[:, :, at]      # [H, nb, 64, D]
    x = raw.view(codes.dtype).float() * scale[l, :, b0:b1, None, None]
    return x.reshape(H, (b1 - b0) * BLOCK, -1)[:, first - b0 * BLOCK : first - b0 * BLOCK + n].transpose(0, 1)


def _ascending(seg_start: Tensor, rows: int) -> list[int]:
    seg = seg_start.tolist()
    if any(b < a for a, b in zip(seg[:-1], seg[1:])) or seg[0] != 0 or seg[-1] > rows:
        raise ValueError(f"seg_start must ascend from 0 within the {rows} rows, got {seg}")
    return seg


def _bounds(cache: KV8Cache, seg_start: Tensor, start: Tensor, rows: int) -> tuple[list[int], list[int]]:
    seg, at = _ascending(seg_start, rows), start.tolist()
    for l, s in enumerate(at):
        n = seg[l + 1] - seg[l]
        if n and (s < 0 or s + n > cache.capacity):
            raise ValueError(f"list {l}: entries {s} .. {s + n} exceed the key/value cache of {cache.capacity} entries per list")
    return seg, at


def kv8_append(cache: KV8Cache, k: Tensor, v: Tensor, seg_start: Tensor, start: Tensor, max_rows: int = 1) -> None:
    """Append the packed rows ``k, v [rows, H, head_dim]`` to their lists, list ``l`` from entry ``start[l]`` on.

    Blocks that receive rows are quantised anew; entries from ``start[l] + n`` on are gone. ``start[l]`` may lie before the
    list's end: at most 64 entries below the greatest length that the list has had (the originals of older blocks are
    gone), or anywhere if it is a multiple of 64. Rows behind
    ``seg_start[-1]`` are ignored. ``k`` and ``v`` may be views (any row and head strides). ``max_rows`` says how many
    rows a list brings at most and only steers speed. A list that would exceed the capacity is an error: raised
    here on the CPU; on a GPU its rows are dropped and the device status word is set (``ops._lib.check_status``).
    """

    check_append(cache, k, v, seg_start, start, max_rows)
    seg, at = _bounds(cache, seg_start, start, k.shape[0])
    for l, s in enumerate(at):
        n = seg[l + 1] - seg[l]
        if n == 0:
            continue
        b0, last = s // BLOCK, (s + n - 1) // BLOCK
        for which, rows, held in (("k", k, cache.k_open), ("v", v, cache.v_open)):
            x = torch.cat([held[l, :, b0 % 2, : s % BLOCK].transpose(0, 1), rows[seg[l] : seg[l + 1]]])
            for b in range(b0, last + 1):
                _store_block(cache, which, l, b, x[(b - b0) * BLOCK : (b - b0 + 1) * BLOCK])
            for b in range(max(b0, last - 1), last + 1):
                part = x[(b - b0) * BLOCK : (b - b0 + 1) * BLOCK]
                held[l, :, b % 2, : part.shape[0]] = part.transpose(0, 1)


def kv8_truncate(cache: KV8Cache, lengths: Tensor) -> None:
    """Make every list end at ``lengths[l]`` entries: a partly filled last block is quantised again from its first
    ``lengths[l] % 64`` originals, so nothing of the dropped entries remains in its scales. How far a list can
    step back is said in :func:`kv8_append`. Lists whose length did not change stay as they are.
    """

    check_index(lengths, cache.lists, "lengths", cache.device)
    for l, n in enumerate(lengths.tolist()):
        if not 0 <= n <= cache.capacity:
            raise ValueError(f"list {l}: length {n} is outside the key/value cache of {cache.capacity} entries per list")
        if n % BLOCK:
            for which, held in (("k", cache.k_open), ("v", cache.v_open)):
                _store_block(cache, which, l, n // BLOCK, held[l, :, n // BLOCK % 2, : n % BLOCK].transpose(0, 1))


def kv8_read(cache: KV8Cache, seg_start: Tensor, start: Tensor, rows: int, dtype: torch.dtype = torch.float32,
             max_rows: int = BLOCK) -> tuple[Tensor, Tensor]:
    """The values that stand in the cache: keys and values ``[rows, H, head_dim]`` of entries ``start[l] .. start[l] + n``
    of every list, packed by ``seg_start``; rows behind ``seg_start[-1]`` are zeros. ``max_rows`` only steers speed."""

    check_read(cache, seg_start, start, rows, dtype, max_rows)
    seg, at = _bounds(cache, seg_start, start, rows)
    out = []
    for which in ("k", "v"):
        x = torch.zeros(rows, cache.heads, cache.head_dim, dtype=dtype, device=cache.device)
        for l, s in enumerate(at):
            x[seg[l] : seg[l + 1]] = _load_entries(cache, which, l, s, seg[l + 1] - seg[l]).to(dtype)
        out.append(x)
    return out[0], out[1]


def kv8_attention(q: Tensor, cache: KV8Cache, seg_start: Tensor, lengths: Tensor, scale: float, max_rows: int = 1,
                  out: Tensor | None = None) -> Tensor:
    """Causal attention of packed new rows over the cache.

    ``q [rows, Hq, head_dim]`` (bf16, fp16 or fp32; ``Hq`` a multiple of the cache's heads, query head ``h`` reads key
    head ``h * H // Hq``). ``lengths [L]`` counts the entries of each list with the new rows' own among them, so row
    ``a`` of the ``n`` rows of list ``l`` sees the first ``lengths[l] - (n - 1 - a)`` entries. Softmax of
    ``scale * q . k`` with fp32 sums, output in ``q.dtype``; a row that sees nothing gives zeros. (The kernel's products take
    fp16 numbers: one for a 16-bit query element, two, 22 bits, for an fp32 one; one for a weight whose output is bf16, 11
    bits and no less than 2^-32 of the row's largest, two for the others.) Rows behind ``seg_start[-1]``
    are left as they are in ``out`` (which may be ``q`` itself, but must not overlap it otherwise) and are zeros without
    it. ``max_rows`` (how many rows a list brings at most) only steers speed. ``lengths`` beyond the capacity count as the
    capacity and are reported like in :func:`kv8_append`, and so are bounds that do not ascend from 0; rows that no list with
    valid bounds covers are zeros. Rows whose codes a kernel waited for in vain are NaN, and reported.
    """

    check_attention(q, cache, seg_start, lengths, scale, max_rows, out)
    seg, size = _ascending(seg_start, q.shape[0]), lengths.tolist()
    out = torch.zeros_like(q, memory_format=torch.contiguous_format) if out is None else out
    group = q.shape[1] // cache.heads
    for l, length in enumerate(size):
        n = seg[l + 1] - seg[l]
        if n == 0:
            continue
        if length > cache.capacity:
            raise ValueError(f"list {l}: length {length} exceeds the key/value cache of {cache.capacity} entries per list")
        k, v = (_load_entries(cache, w, l, 0, max(length, 0)).transpose(0, 1) for w in ("k", "v"))     # [H, n, D]
        x = q[seg[l] : seg[l + 1]].float().view(n, cache.heads, group, -1).permute(1, 0, 2, 3)         # [H, n, group, D]
        s = torch.einsum("hagd,hed->hage", x, k) * scale
        hidden = torch.arange(k.shape[1], device=q.device) >= (length - (n - 1 - torch.arange(n, device=q.device))).unsqueeze(1)
        s = s.masked_fill(hidden.view(1, n, 1, -1), float("-inf"))
        p = torch.softmax(s, dim=-1).masked_fill(hidden.view(1, n, 1, -1), 0.0)                        # (no entry: NaN -> 0)
        o = torch.einsum("hage,hed->hagd", p, v)
        out[seg[l] : seg[l + 1]] = o.permute(1, 0, 2, 3).reshape(n, q.shape[1], -1).to(q.dtype)
    return out


# ------------------------------------------------------------------------------------- statement: verification
def verify_draft(target_probs: Tensor, draft_tokens: Tensor, draft_probs: Tensor | None, accept_u: Tensor, sample_u: Tensor,
                 draft_len: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """Verify drafted tokens and draw the token after them: ``(accepted [B] int32, token [B] int32)``.

    ``target_probs [B, n + 1, V]``: the target's probabilities at the positions of the ``n`` drafted tokens and after
    them (rows need not sum to exactly one). ``draft_probs [B, n, V]``: what each token of ``draft_tokens [B, n]`` was
    drawn from, ``None`` if each was the draft's certain choice. ``accept_u [B, n]``, ``sample_u [B]``: uniform numbers in
    ``[0, 1)``. ``draft_len [B]``: drafted tokens of each sequence (the rest is padding and not looked at).

    Token ``i`` is accepted while ``u_i q_i(x_i) < p_i(x_i)`` (fp32 product). With ``a`` accepted, the next token is the
    lowest ``j`` with ``r_0 + .. + r_j > w * sum(r)``, summed in 64 bits, where ``r = p_len`` if all were accepted and
    otherwise ``r = max(p_a - q_a, 0)`` (``p_a`` without ``x_a`` where there are no ``draft_probs``), or ``p_a`` if that
    leaves nothing. ``-1`` if ``p_a`` has no mass either. Values below ``2^-126`` and NaN count as zero,
    tokens outside the vocabulary as refused.
    """

    check_verify(target_probs, draft_tokens, draft_probs, accept_u, sample_u, draft_len)
    B, n, V = target_probs.shape[0], draft_tokens.shape[1], target_probs.shape[2]
    dev = target_probs.device
    flush = lambda t: torch.where(t >= 2.0 ** -126, t, 0.0)              # noqa: E731  (NaN -> 0)
    x = draft_tokens.long()
    known = (x >= 0) & (x < V)
    at = x.clamp(0, V - 1).unsqueeze(-1)
    length = torch.full((B,), n, device=dev) if draft_len is None else draft_len.long().clamp(0, n)
    px = torch.where(known, flush(target_probs[:, :n].gather(2, at).squeeze(-1).float()), 0.0)
    qx = torch.ones_like(px) if draft_probs is None else torch.where(known, flush(draft_probs.gather(2, at).squeeze(-1).float()), 0.0)
    ok = (accept_u * qx < px) & (torch.arange(n, device=dev) < length.unsqueeze(1))
    a = ok.long().cumprod(dim=1).sum(dim=1)
    b = torch.arange(B, device=dev)
    r = flush(target_probs[b, a].float())
    if n > 0:
        i = a.clamp(max=n - 1)
        if draft_probs is None:
            rest = torch.where(torch.arange(V, device=dev) == x[b, i].unsqueeze(1), 0.0, r)
        else:
            rest = flush(r - flush(draft_probs[b, i].float()))
        use = (a < length) & (rest > 0).any(dim=1)
        r = torch.where(use.unsqueeze(1), rest, r)
    run = r.double().cumsum(dim=1)
    hit = (run > sample_u.double().unsqueeze(1) * run[:, -1:]) & (r > 0)
    last = V - 1 - (r > 0).flip(1).int().argmax(dim=1)                   # (rounding left none: the last one with mass)
    token = torch.where(hit.any(dim=1), hit.int().argmax(dim=1), torch.where((r > 0).any(dim=1), last, -1))
    return a.to(torch.int32), token.to(torch.int32)
