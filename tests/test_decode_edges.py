"""The decoding ops and decode states at the edges: waits that run out, row bounds, threads, other callers' decode states."""

import pytest
import torch

from nestor_b200 import ops

DEV = "cuda"


def i32(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def seg_of(counts, device="cpu"):
    return i32([0, *torch.tensor(counts).cumsum(0).tolist()], device)


def random_cache(L, H, blocks, hd, code, seed, kind=torch.bfloat16):
    """Any codes and scales, whole blocks (no NaN code among them)."""

    g = torch.Generator(DEV).manual_seed(seed)
    codes = [torch.randint(-127, 128, (L, H, blocks, -(-hd // 8), 512), generator=g, device=DEV, dtype=torch.int8) for _ in range(2)]
    if code != torch.int8:
        codes = [torch.where((c & 0x7F) == 0x7F, 0, c).view(code) for c in codes]
    scale = [torch.rand(L, H, blocks, generator=g, device=DEV) * 0.02 for _ in range(2)]
    held = [torch.zeros(L, H, 2, 64, hd, device=DEV, dtype=kind) for _ in range(2)]
    return ops.KV8Cache(*codes, *scale, *held)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("shape", [
    (6, 2, 8, 40, 1, [1, 1, 0, 1, 1, 1]),             # by tasks
    (5, 2, 8, 104, 2, [3, 1, 1, 0, 5]),               # by tasks, wide heads, two column tiles
    (3, 2, 400, 40, 1, [1, 1, 1]),                    # by units, one for a warp
    (3, 4, 400, 128, 2, [5, 0, 2]),
    (96, 4, 420, 16, 1, [1] * 96),                    # by units, fetched at run time
    (24, 4, 420, 104, 4, [5] * 24),
], ids=lambda s: f"{s[0]}x{s[2]}-h{s[1]}x{s[4]}-d{s[3]}")
def test_a_wait_for_codes_that_runs_out_is_reported_and_leaves_nan(shape, code, monkeypatch):
    """The waits of the attention are given no time at all: the call returns, the status says so, no row looks computed,
    rows that no list brings are as ever, and the next call is right."""

    from nestor_b200.ops import _lib, cuda_decode
    L, H, blocks, hd, group, counts = shape
    dev = torch.device(DEV, 0)
    cache = random_cache(L, H, blocks, hd, code, 3)
    rows = sum(counts)
    q = torch.randn(rows + 2, H * group, hd, device=DEV).bfloat16()
    seg, lengths = seg_of(counts, DEV), i32([blocks * 64 - 7 * (l % 5) for l in range(L)], DEV)
    want = ops.kv8_attention(q, cache, seg, lengths, 0.05, max_rows=max(counts))
    _lib.check_status(dev)
    monkeypatch.setattr(cuda_decode, "WAIT_POLLS", 0)
    got = ops.kv8_attention(q, cache, seg, lengths, 0.05, max_rows=max(counts))
    with pytest.raises(RuntimeError, match="wait gave up"):
        _lib.check_status(dev)
    assert got[:rows].isnan().all() and (got[rows:] == 0).all()
    given = torch.full_like(q, 3.0)
    ops.kv8_attention(q, cache, seg, lengths, 0.05, max_rows=max(counts), out=given)
    with pytest.raises(RuntimeError, match="wait gave up"):
        _lib.check_status(dev)
    assert given[:rows].isnan().all() and (given[rows:] == 3).all()
    monkeypatch.undo()
    assert torch.equal(want, ops.kv8_attention(q, cache, seg, lengths, 0.05, max_rows=max(counts)))
    _lib.check_status(dev)
