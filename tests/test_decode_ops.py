"""The decoding ops: 8-bit key/value cache (append, truncate, read, attention) and verification of drafted tokens."""

import copy
import math
import pickle

import pytest
import torch

from nestor_b200 import ops
from nestor_b200.ops import decode as D

CODES = [torch.int8, torch.float8_e4m3fn]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def seg_of(counts, device="cpu"):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=device)


def i32(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def filled(lengths, H, D_, code, kind, seed=0, capacity=None, device="cpu"):
    """A cache whose lists hold ``lengths`` random entries (and the appended rows)."""

    g = torch.Generator().manual_seed(seed)
    cache = ops.kv8_cache(len(lengths), H, capacity or max(1, *lengths), D_, device, code, kind)
    rows = sum(lengths)
    k = (torch.randn(rows, H, D_, generator=g) * torch.rand(rows, 1, 1, generator=g).exp()).to(kind).to(device)
    v = torch.randn(rows, H, D_, generator=g).to(kind).to(device)
    ops.kv8_append(cache, k, v, seg_of(lengths, device), i32([0] * len(lengths), device), max_rows=max(1, *lengths))
    return cache, k, v


def same(a, b):
    """Bit-equal caches (NaN scales included)."""

    raw = lambda t: t.contiguous().view(torch.uint8).cpu()       # noqa: E731
    return all(torch.equal(raw(getattr(a, f)), raw(getattr(b, f))) for f in ("k_codes", "v_codes", "k_scale", "v_scale"))


def to(cache, device):
    return D.KV8Cache(*(getattr(cache, f).to(device) for f in ("k_codes", "v_codes", "k_scale", "v_scale", "k_open", "v_open")))


def values64(cache, which, l, n):
    """Entries ``0 .. n`` of list ``l`` in 64 bits, ``[H, n, D]``, from the codes and the layout's definition."""

    codes, scale = (cache.k_codes, cache.k_scale) if which == "k" else (cache.v_codes, cache.v_scale)
    _, H, nb, U, _ = codes.shape
    raw = codes[l].view(torch.uint8).view(H, nb, U, 8, 4, 4, 2, 2)            # g, t, m, h, i
    order = (0, 1, 5, 6, 3, 2, 4, 7) if which == "k" else (0, 1, 5, 6, 4, 7, 2, 3)
    x = raw.permute(*order).reshape(H, nb, 64, 8 * U).view(codes.dtype).double()
    return (x * scale[l].double()[..., None, None]).reshape(H, nb * 64, 8 * U)[:, :n, : cache.head_dim]


def attention64(q, cache, seg, lengths, scale):
    """Softmax attention in 64 bits and, beside it, what the kernel's arithmetic may be off by.

    With ``S = scale * sum |q k|`` the largest absolute score sum of a row: a score is off by at most the fp32 sums of
    D products, ``(D + 8) 2^-23 S``, and the exponential by 2^-22 and the rounding of its argument, ``2^-23 (|s| +
    |max|) log2(e)``; a weight is rounded to fp16 (2^-11; 2^-21 where it is split in two). Relative errors ``e`` of the
    weights move their normalised mixture by at most ``2 e vmax``; the fp32 sums over ``n`` entries add
    ``(n / 16 + 16) 2^-23 vmax``; the output is rounded by half a step of its type.
    """

    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[1] // cache.heads
    half = torch.finfo(q.dtype).eps / 2
    lift = 128.0 if q.dtype != torch.float32 and cache.dtype == torch.int8 else 0.0
    for l, length in enumerate(lengths):
        n = int(seg[l + 1] - seg[l])
        for a in range(n):
            see = length - (n - 1 - a)
            if see <= 0:
                continue
            k, v = (values64(cache, w, l, length)[:, :see].repeat_interleave(group, 0) for w in ("k", "v"))
            x = q[int(seg[l]) + a].double().unsqueeze(1)
            s = (x * k).sum(-1) * scale
            extra = [(lift * t[l].double()).repeat_interleave(64, 1)[:, :see].repeat_interleave(group, 0) for t in (cache.k_scale, cache.v_scale)]
            big = ((x.abs() * (k.abs() + extra[0].unsqueeze(-1))).sum(-1) * scale).amax(-1)
            p = torch.softmax(s, -1)
            o = (p.unsqueeze(-1) * v).sum(1)
            e = big * (q.shape[2] + 8) * 2.0 ** -23 + 2.0 ** -22 + 2 * s.abs().amax(-1) * 1.45 * 2.0 ** -23
            e = torch.expm1(2 * e) + (2.0 ** -21 if q.dtype == torch.float32 else 2.0 ** -11)
            vmax = v.abs().amax(dim=(1, 2))
            out[int(seg[l]) + a] = o
            tol[int(seg[l]) + a] = (2 * e * vmax + (see / 16 + 16) * 2.0 ** -23 * (vmax + extra[1].amax(-1))).unsqueeze(-1) + half * o.abs() * 1.01
    return out, tol


def check_attention(q, cache, seg, lengths, scale, got):
    host = to(cache, "cpu")
    want, tol = attention64(q.cpu(), host, seg.cpu(), lengths, scale)
    n = int(seg[-1])
    off = (got[:n].double().cpu() - want[:n]).abs()
    assert not torch.isnan(got).any()
    assert (off <= tol[:n]).all(), f"off by {(off / tol[:n].clamp_min(1e-300)).max():.3g} times the bound"


# ------------------------------------------------------------------------------------------------- cache, statement
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hd", [5, 40, 128])
def test_codes_stand_for_the_appended_values(code, hd):
    cache, k, v = filled([70, 0, 1, 64], 3, hd, code, torch.float32, seed=1)
    assert cache.capacity == 128 and cache.head_dim == hd
    step = 2.0 ** -4 if code == torch.float8_e4m3fn else 0.0      # half a step, relative to the value
    back = ops.kv8_read(cache, seg_of([70, 0, 1, 64]), i32([0, 0, 0, 0]), 140)
    for x, y, which in ((k, back[0], "k"), (v, back[1], "v")):
        assert torch.equal(y[135:], torch.zeros(5, 3, hd))        # rows behind the last list
        for l, (a, n) in enumerate(((0, 70), (70, 0), (70, 1), (71, 64))):
            held = values64(cache, which, l, n).transpose(0, 1)
            assert torch.allclose(y[a : a + n].double(), held, rtol=2.0 ** -23, atol=0)
            for b in range(0, n, 64):
                block = x[a + b : min(a + b + 64, a + n)].double()
                amax = block.abs().amax(dim=(0, 2), keepdim=True)
                # int8: half of amax / 127; e4m3: half a step of the value, or of the smallest exponent (2^-9 of 448)
                tol = amax / 254 if code == torch.int8 else torch.maximum(block.abs() * step, amax / 448 * 2.0 ** -10)
                assert ((block - held[b : b + 64]).abs() <= tol * (1 + 1e-6)).all()


@pytest.mark.parametrize("code", CODES)
def test_a_block_is_a_function_of_its_contents(code):
    """Appending row by row, in pieces or at once, with steps back in between, leaves the same codes and scales."""

    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(150, 2, 24, generator=g), torch.randn(150, 2, 24, generator=g)
    k[100] *= 50                                                  # a late outlier rescales its block
    whole = ops.kv8_cache(1, 2, 192, 24, dtype=code, open_dtype=torch.float32)
    ops.kv8_append(whole, k, v, seg_of([150]), i32([0]))
    pieces = ops.kv8_cache(1, 2, 192, 24, dtype=code, open_dtype=torch.float32)
    at = 0
    for n in (1, 62, 1, 30, 40, 16):
        if at + n < 150:                                          # rows that are refused and taken back
            wrong = torch.full((40, 2, 24), 99.0)
            ops.kv8_append(pieces, wrong, wrong, seg_of([40]), i32([at]))
            ops.kv8_truncate(pieces, i32([at]))
        ops.kv8_append(pieces, k[at : at + n], v[at : at + n], seg_of([n]), i32([at]))
        at += n
    assert at == 150
    for f in ("k_scale", "v_scale"):
        assert torch.equal(getattr(whole, f)[..., :3], getattr(pieces, f)[..., :3])
    assert torch.equal(whole.k_codes[:, :, :3].view(torch.uint8), pieces.k_codes[:, :, :3].view(torch.uint8))
    assert torch.equal(whole.v_codes[:, :, :3].view(torch.uint8), pieces.v_codes[:, :, :3].view(torch.uint8))
    # a step back across a block's border
    ops.kv8_truncate(pieces, i32([120]))
    short = ops.kv8_cache(1, 2, 192, 24, dtype=code, open_dtype=torch.float32)
    ops.kv8_append(short, k[:120], v[:120], seg_of([120]), i32([0]))
    assert torch.equal(short.k_scale[..., :2], pieces.k_scale[..., :2])
    assert torch.equal(short.k_codes[:, :, :2].view(torch.uint8), pieces.k_codes[:, :, :2].view(torch.uint8))


@pytest.mark.parametrize("code", CODES)
def test_blocks_of_zeros_infinities_and_tiny_values(code):
    k = torch.zeros(5, 1, 8)
    k[1:, 0, 0] = torch.tensor([1e-38, math.inf, math.nan, 2.0])
    cache = ops.kv8_cache(5, 1, 64, 8, dtype=code, open_dtype=torch.float32)
    ops.kv8_append(cache, k, k, seg_of([1] * 5), i32([0] * 5))
    assert cache.k_scale[:2, 0, 0].tolist() == [0.0, 0.0] and cache.k_scale[2:4].isnan().all() and not cache.k_scale[4].isnan()
    back, _ = ops.kv8_read(cache, seg_of([1] * 5), i32([0] * 5), 5)
    assert torch.equal(back[:2], torch.zeros(2, 1, 8)) and back[2:4].isnan().all() and back[4, 0, 0] == 2.0


@pytest.mark.parametrize("kind", TYPES)
def test_statement_of_attention_matches_64_bits(kind):
    lengths, counts = [130, 3, 64, 0, 7], [3, 1, 0, 2, 7]
    cache, _, _ = filled(lengths, 2, 20, torch.int8, kind, seed=4)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(15, 6, 20, generator=g).to(kind)
    seg = seg_of(counts)
    got = ops.kv8_attention(q, cache, seg, i32(lengths), 0.3)
    check_attention(q, cache, seg, lengths, 0.3, got)
    assert torch.equal(got[4:6], torch.zeros_like(got[4:6]))      # an empty list
    assert torch.equal(got[13:], torch.zeros_like(got[13:]))      # behind the last list
    given = torch.full_like(q, 7.0)
    assert ops.kv8_attention(q, cache, seg, i32(lengths), 0.3, out=given) is given
    assert torch.equal(given[:13], got[:13]) and (given[13:] == 7.0).all()


def test_refusals():
    cache = ops.kv8_cache(2, 3, 100, 16)
    seg, start = seg_of([1, 1]), i32([0, 0])
    row = torch.zeros(2, 3, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="int8 or float8"):
        ops.kv8_cache(1, 1, 1, 8, dtype=torch.uint8)
    with pytest.raises(ValueError, match="head_dim"):
        ops.kv8_cache(1, 1, 1, 129)
    with pytest.raises(ValueError, match="unlike shapes"):
        ops.KV8Cache(cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale[:1], cache.k_open, cache.v_open)
    with pytest.raises(AttributeError, match="fixed"):
        cache.k_scale = cache.v_scale
    with pytest.raises(ValueError, match="scales are float32"):
        ops.KV8Cache(cache.k_codes, cache.v_codes, cache.k_scale.double(), cache.v_scale.double(), cache.k_open, cache.v_open)
    with pytest.raises(ValueError, match="k must be"):
        ops.kv8_append(cache, row.float(), row, seg, start)
    with pytest.raises(ValueError, match="of keys but"):
        ops.kv8_append(cache, row, row[:1], seg, start)
    with pytest.raises(ValueError, match="seg_start must be"):
        ops.kv8_append(cache, row, row, seg.long(), start)
    with pytest.raises(ValueError, match="start must be"):
        ops.kv8_append(cache, row, row, seg, start[:1])
    with pytest.raises(ValueError, match="max_rows"):
        ops.kv8_append(cache, row, row, seg, start, max_rows=0)
    with pytest.raises(ValueError, match="exceed the key/value cache"):
        ops.kv8_append(cache, row, row, seg, i32([0, 128]))
    with pytest.raises(ValueError, match="ascend"):
        ops.kv8_append(cache, row, row, i32([0, 2, 1]), start)
    with pytest.raises(ValueError, match="ascend"):
        ops.kv8_append(cache, row, row, i32([0, 1, 3]), start)
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.kv8_append(cache, row.clone().requires_grad_(), row, seg, start)
    with pytest.raises(ValueError, match="outside the key/value cache"):
        ops.kv8_truncate(cache, i32([0, 129]))
    with pytest.raises(ValueError, match="kv8_read writes"):
        ops.kv8_read(cache, seg, start, 2, dtype=torch.int8)
    with pytest.raises(ValueError, match="rows must be in"):
        ops.kv8_read(cache, seg, start, -1)
    for q in (row[:, :2], row[..., :8], row.double()):
        with pytest.raises(ValueError, match="q must be"):
            ops.kv8_attention(q, cache, seg, start, 1.0)
    with pytest.raises(ValueError, match="scale"):
        ops.kv8_attention(row, cache, seg, start, 0.0)
    for out in (row.float(), row[:1].expand(2, 3, 16), torch.zeros(2, 3, 32, dtype=torch.bfloat16)[..., ::2]):
        with pytest.raises(ValueError, match="out must"):
            ops.kv8_attention(row, cache, seg, start, 1.0, out=out)
    with pytest.raises(ValueError, match="16-byte"):
        odd = torch.zeros(cache.k_codes.numel() + 1, dtype=torch.int8)[1:].view(cache.k_codes.shape)
        ops.KV8Cache(odd, cache.v_codes, cache.k_scale, cache.v_scale, cache.k_open, cache.v_open)
    with pytest.raises(ValueError, match="exceeds the key/value cache"):
        ops.kv8_attention(row, cache, seg, i32([0, 129]), 1.0)
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.kv8_attention(row.clone().requires_grad_(), cache, seg, start, 1.0)
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.kv8_attention(row, cache, seg, start, 1.0, out=row.clone().requires_grad_())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_copies_of_a_cache_go_their_own_way(device):
    cache = ops.kv8_cache(2, 3, 100, 16, device)
    rows = [torch.randn(4, 3, 16, device=device).bfloat16() for _ in range(2)]
    seg, at = torch.tensor([0, 2, 4], dtype=torch.int32, device=device), torch.zeros(2, dtype=torch.int32, device=device)
    ops.kv8_append(cache, *rows, seg, at, max_rows=2)
    twins = copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))
    before = [t.clone() for t in ops.kv8_read(cache, seg, at, 4)]
    ops.kv8_append(cache, -rows[0], -rows[1], seg, at, max_rows=2)
    for twin in twins:
        assert twin.k_codes.data_ptr() != cache.k_codes.data_ptr() and twin.device == cache.device
        for x, y, z in zip(before, ops.kv8_read(twin, seg, at, 4), ops.kv8_read(cache, seg, at, 4)):
            assert torch.equal(x, y) and torch.equal(x, -z)


@pytest.mark.gpu
@pytest.mark.parametrize("capacity", [1024, 300_000])             # by tasks; by units with a workspace
def test_attention_into_its_own_queries(capacity):
    n = 700
    cache = ops.kv8_cache(2, 2, capacity, 40, "cuda")
    seg = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(2 * n, 2, 40, device="cuda").bfloat16() for _ in range(2))
    ops.kv8_append(cache, k, v, seg, torch.zeros(2, dtype=torch.int32, device="cuda"), max_rows=n)
    q = torch.randn(6, 4, 40, device="cuda").bfloat16()
    few, lengths = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda"), torch.tensor([n, n - 60], dtype=torch.int32, device="cuda")
    want = ops.kv8_attention(q, cache, few, lengths, 1 / 40, max_rows=3)
    own = q.clone()
    assert ops.kv8_attention(own, cache, few, lengths, 1 / 40, max_rows=3, out=own) is own
    assert torch.equal(own[:5], want[:5]) and torch.equal(own[5:], q[5:])


def test_argument_blocks_match_the_built_library():
    """The ctypes mirrors have the sizes of the C structures (8-byte pointers and longs, 4-byte ints)."""

    import ctypes as C
    from nestor_b200.ops import cuda_decode as K
    assert C.sizeof(K.CacheArgs) == 7 * 8 + 7 * 4 + 4
    assert C.sizeof(K.RowArgs) == 8 * 8 + 2 * 8 + 2 * 4
    assert C.sizeof(K.AttentionArgs) == 8 * 8 + 6 * 4
    assert C.sizeof(K.VerifyArgs) == 12 * 8 + 5 * 4 + 4


# ---------------------------------------------------------------------------------------------- verification, statement
def verify64(p, x, q, u, w, lens):
    """The definition, sequence by sequence, in 64 bits."""

    import numpy as np
    accepted, token = [], []
    flush = lambda t: torch.where(t.double() >= 2.0 ** -126, t.double(), 0.0)       # noqa: E731
    for b in range(p.shape[0]):
        a = 0
        while a < lens[b]:
            t = int(x[b, a])
            known = 0 <= t < p.shape[2]
            px = float(flush(p[b, a, t])) if known else 0.0
            qx = 1.0 if q is None else (float(flush(q[b, a, t])) if known else 0.0)
            if not float(np.float32(float(u[b, a])) * np.float32(qx)) < px:
                break
            a += 1
        r = flush(p[b, a])
        if a < lens[b]:
            rest = r.clone()
            if q is None:
                if 0 <= int(x[b, a]) < p.shape[2]:
                    rest[int(x[b, a])] = 0
            else:
                rest = (r - flush(q[b, a])).clamp_min(0)
            if (rest > 0).any():
                r = rest
        run = r.cumsum(0)
        hit = ((run > float(w[b]) * run[-1]) & (r > 0)).nonzero()
        some = (r > 0).nonzero()
        accepted.append(a)
        token.append(int(hit[0]) if len(hit) else (int(some[-1]) if len(some) else -1))
    return accepted, token


def drafts(B, n, V, kind, greedy, seed):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(B, n + 1, V, generator=g) * 2
    p = torch.softmax(z, -1).to(kind)
    near = z[:, :n] + torch.randn(B, n, V, generator=g) * 0.5
    if greedy:
        q, x = None, near.argmax(-1)
    else:
        q = torch.softmax(near, -1).to(kind)
        x = torch.multinomial(q.float().view(-1, V), 1, generator=g).view(B, n) if n else torch.zeros(B, 0, dtype=torch.long)
    u, w = torch.rand(B, n, generator=g), torch.rand(B, generator=g)
    if greedy:
        u *= 0.3
    return p, x, q, u, w, torch.randint(0, n + 1, (B,), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("greedy", [False, True])
def test_statement_of_verification(kind, greedy):
    for n in (0, 1, 5):
        p, x, q, u, w, lens = drafts(13, n, 31, kind, greedy, n)
        for use in (lens, None):
            a, t = ops.verify_draft(p, x, q, u, w, use)
            want = verify64(p, x, q, u, w, [n] * 13 if use is None else use.tolist())
            assert (a.tolist(), t.tolist()) == want


def edge_cases():
    """``(p, x, q, u, w, accepted, token)`` at the borders of the definition."""

    p = torch.tensor([[[0.5, 0.5, 0.0, 0.0], [0.0, 0.25, 0.0, 0.75]]])
    one = lambda x, q, u, w: (p, torch.tensor([[x]]), None if q is None else torch.tensor([[q]]), torch.tensor([[u]]), torch.tensor([w]))   # noqa: E731
    return [
        (*one(0, [1.0, 0.0, 0.0, 0.0], 0.4999, 0.0), 1, 1),          # accepted; the draw at zero skips entries without mass
        (*one(0, [1.0, 0.0, 0.0, 0.0], 0.5, 0.99), 0, 1),            # u q = p is a refusal; only token 1 remains
        (*one(2, [0.0, 0.0, 1.0, 0.0], 0.0, 0.6), 0, 1),             # the target gives the drafted token nothing
        (*one(0, [0.9, 0.9, 0.9, 0.9], 0.99, 0.5), 0, 1),            # the rest is empty: p itself, 0.5 is not above 0.5
        (*one(0, None, 0.5, 0.3), 0, 1),                             # a certain draft that is refused leaves p without it
        (*one(0, None, 0.4999, 0.25), 1, 3),                         # accepted; 0.25 of the mass is not above 0.25
        (*one(-1, None, 0.0, 0.0), 0, 0),                            # no such token
        (*one(9, [1.0, 0.0, 0.0, 0.0], 0.0, 0.0), 0, 1),
        (*one(0, None, 0.1, 1.0), 1, 3),                             # out of range: the last entry with mass
        (p * 0, torch.tensor([[1]]), None, torch.tensor([[0.0]]), torch.tensor([0.5]), 0, -1),        # no mass at all
        (torch.tensor([[[0.5, math.nan, 0.5, 0.0], [0.0, 0.25, 0.0, 0.75]]]), torch.tensor([[1]]), torch.tensor([[[0.6, 0.2, math.nan, 0.0]]]),
         torch.tensor([[0.1]]), torch.tensor([0.9]), 0, 2),          # a NaN in p is refused, one in q takes nothing off
        (torch.tensor([[[0.5, 0.0, 0.5, 0.0], [0.0, 0.25, 0.0, 0.75]]]), torch.tensor([[2]]), torch.tensor([[[0.6, 0.2, math.nan, 0.0]]]),
         torch.tensor([[0.1]]), torch.tensor([0.2]), 1, 1),
        (torch.full_like(p, math.nan), torch.tensor([[1]]), None, torch.tensor([[0.0]]), torch.tensor([0.5]), 0, -1),
    ]


def test_borders_of_verification():
    for p, x, q, u, w, accepted, token in edge_cases():
        a, t = ops.verify_draft(p, x, q, u, w)
        assert (a.tolist(), t.tolist()) == ([accepted], [token])


@pytest.mark.parametrize("greedy", [False, True])
def test_verified_tokens_are_distributed_as_the_target(greedy):
    """Over a grid of both random numbers and the draft's own choice, the first token after verification has the
    target's distribution: midpoint sums of step functions with at most 2 V borders are off by at most 2 V / 400."""

    p = torch.tensor([0.1, 0.35, 0.05, 0.3, 0.2])
    q = torch.tensor([0.3, 0.1, 0.2, 0.3, 0.1]) if not greedy else torch.tensor([0.0, 0.0, 0.0, 1.0, 0.0])
    grid = (torch.arange(400) + 0.5) / 400
    u, w = torch.meshgrid(grid, grid, indexing="ij")
    u, w = u.reshape(-1), w.reshape(-1)
    got = torch.zeros(5, dtype=torch.float64)
    for x in range(5):
        if q[x] == 0:
            continue
        B = u.numel()
        target = p.expand(B, 2, 5)
        a, t = ops.verify_draft(target, torch.full((B, 1), x), None if greedy else q.expand(B, 1, 5), u.unsqueeze(1), w)
        first = torch.where(a == 1, x, t.long())
        got += float(q[x]) * torch.bincount(first, minlength=5).double() / B
    assert (got - p.double()).abs().max() <= 10 / 400


def test_verification_refusals():
    p, x, q, u, w, lens = drafts(3, 2, 7, torch.float32, False, 0)
    for bad in ((p[0], x, q, u, w), (p.double(), x, q, u, w), (p, x[:, :1], q, u, w), (p, x.float(), q, u, w), (p, x, q[:, :1], u, w),
                (p, x, q.half(), u, w), (p, x, q, u.double(), w), (p, x, q, u, w[:2])):
        with pytest.raises(ValueError, match="verify_draft"):
            ops.verify_draft(*bad)
    with pytest.raises(ValueError, match="draft_len"):
        ops.verify_draft(p, x, q, u, w, lens.long())
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.verify_draft(p.clone().requires_grad_(), x, q, u, w)


# ------------------------------------------------------------------------------------------------------- kernels
DEV = "cuda"


def strided(x):
    """The same rows inside a wider buffer (as the key range of a fused projection output is)."""

    rows, H, hd = x.shape
    wide = torch.full((rows, 2 * H * hd + 3), math.nan, dtype=x.dtype, device=x.device)
    wide[:, 3 : 3 + H * hd] = x.reshape(rows, -1)
    return wide[:, 3 : 3 + H * hd].view(rows, H, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd", [1, 8, 30, 40, 60, 100, 128])
def test_append_truncate_read_kernels(code, kind, hd):
    g = torch.Generator().manual_seed(hd)
    L, H = 6, 3
    host = ops.kv8_cache(L, H, 500, hd, "cpu", code, kind)
    dev = to(host, DEV)
    at = [0, 0, 0, 0, 0, 0]
    # a prompt, single rows, several rows over a block's border, steps back, a chunk at a border, nothing
    rounds = [([200, 0, 64, 1, 63, 0], 0), ([1, 1, 1, 1, 1, 1], 0), ([5, 0, 9, 62, 2, 0], 3), ([60, 64, 1, 0, 30, 0], 40), ([0] * 6, 0)]
    for i, (counts, back) in enumerate(rounds):
        if back:
            at = [max(0, a - back) for a in at]
            ops.kv8_truncate(host, i32(at))
            ops.kv8_truncate(dev, i32(at, DEV))
            assert same(host, dev)
        rows = sum(counts) + 2                                    # two rows behind the last list
        k, v = (torch.randn(rows, H, hd, generator=g) * 3).to(kind), torch.randn(rows, H, hd, generator=g).to(kind)
        args = seg_of(counts), i32(at)
        ops.kv8_append(host, k, v, *args, max_rows=max(1, *counts))
        kd, vd = k.to(DEV), v.to(DEV)
        if i % 2:
            kd, vd = strided(kd), strided(vd)
        ops.kv8_append(dev, kd, vd, *(t.to(DEV) for t in args), max_rows=max(1, *counts) if i != 2 else 1)
        assert same(host, dev), (i, counts)
        at = [a + n for a, n in zip(at, counts)]
        for out in TYPES:
            first = [a // 2 for a in at]
            part = [a - f for a, f in zip(at, first)]
            want = ops.kv8_read(host, seg_of(part), i32(first), sum(part) + 3, dtype=out)
            got = ops.kv8_read(dev, seg_of(part, DEV), i32(first, DEV), sum(part) + 3, dtype=out, max_rows=1 if i == 1 else 64)
            assert torch.equal(want[0], got[0].cpu()) and torch.equal(want[1], got[1].cpu())
    from nestor_b200.ops import _lib
    _lib.check_status(torch.device(DEV, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_append_kernel_on_zeros_infinities_and_tiny_values(code):
    k = torch.zeros(6, 1, 8)
    k[1:, 0, 0] = torch.tensor([1e-38, math.inf, math.nan, 2.0, -3e38])
    host = ops.kv8_cache(6, 1, 64, 8, "cpu", code, torch.float32)
    dev = to(host, DEV)
    ops.kv8_append(host, k, k, seg_of([1] * 6), i32([0] * 6))
    ops.kv8_append(dev, k.to(DEV), k.to(DEV), seg_of([1] * 6, DEV), i32([0] * 6, DEV))
    assert torch.equal(host.k_codes.view(torch.uint8), dev.k_codes.cpu().view(torch.uint8))
    assert torch.equal(host.k_scale.nan_to_num(-1), dev.k_scale.cpu().nan_to_num(-1))


@pytest.mark.gpu
def test_rows_beyond_the_capacity_are_dropped_and_reported():
    from nestor_b200.ops import _lib
    dev = torch.device(DEV, 0)
    _lib.check_status(dev)
    cache, _, _ = filled([60, 10], 1, 16, torch.int8, torch.bfloat16, capacity=64, device=DEV)
    before = cache.k_codes.clone()
    row = torch.ones(9, 1, 16, dtype=torch.bfloat16, device=DEV)
    ops.kv8_append(cache, row, row, seg_of([8, 1], DEV), i32([60, 10], DEV))
    assert torch.equal(before[0], cache.k_codes[0]) and not torch.equal(before[1], cache.k_codes[1])
    with pytest.raises(RuntimeError, match="capacity"):
        _lib.check_status(dev)
    ops.kv8_attention(row, cache, seg_of([8, 1], DEV), i32([65, 10], DEV), 1.0)
    with pytest.raises(RuntimeError, match="capacity"):
        _lib.check_status(dev)
    for seg in ([0, 4, 12], [0, 3, 2]):                           # past the rows; descending
        ops.kv8_append(cache, row, row, i32(seg, DEV), i32([0, 0], DEV))
        with pytest.raises(RuntimeError, match="capacity"):
            _lib.check_status(dev)
        out = ops.kv8_attention(row, cache, i32(seg, DEV), i32([5, 5], DEV), 1.0)
        assert not out.isnan().any()
        with pytest.raises(RuntimeError, match="capacity"):
            _lib.check_status(dev)
    _lib.check_status(dev)


SHAPES = [
    # lengths, rows, H, group, hd
    ([1], [1], 1, 1, 40),
    ([64, 63, 65, 128, 1, 0], [1, 1, 1, 1, 1, 1], 2, 1, 40),
    ([1000, 40, 0, 333, 129], [1, 0, 0, 1, 1], 5, 1, 40),
    ([700, 5, 64, 70], [5, 5, 1, 9], 3, 1, 60),
    ([257, 2000], [2, 1], 2, 8, 128),
    ([100, 30], [30, 30], 2, 1, 64),
    ([300], [3], 1, 4, 80),
    ([90, 80], [11, 40], 1, 3, 128),
    ([500, 17], [1, 2], 16, 1, 8),
    ([400, 66, 1], [1, 4, 1], 2, 2, 101),
    ([5000], [1], 1, 1, 30),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{len(s[0])}x{max(s[0])}-h{s[2]}x{s[3]}-d{s[4]}")
def test_attention_kernel(shape, code, kind):
    lengths, counts, H, group, hd = shape
    cache, _, _ = filled(lengths, H, hd, code, kind, seed=7, device=DEV)
    g = torch.Generator().manual_seed(8)
    rows = sum(counts)
    q = (torch.randn(rows, H * group, hd, generator=g) * torch.randn(rows, H * group, 1, generator=g).exp() * 3).to(kind).to(DEV)
    seg = seg_of(counts, DEV)
    scale = 1.0 / hd ** 0.5
    got = ops.kv8_attention(q, cache, seg, i32(lengths, DEV), scale, max_rows=max(counts))
    check_attention(q, cache, seg, lengths, scale, got)
    other = ops.kv8_attention(strided(q), cache, seg, i32(lengths, DEV), scale, max_rows=max(counts))
    assert torch.equal(got, other)
    hint = ops.kv8_attention(q, cache, seg, i32(lengths, DEV), scale, max_rows=64)
    check_attention(q, cache, seg, lengths, scale, hint)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_attention_does_not_look_behind_a_list(code):
    """Bytes and scales that no list holds (NaN codes among them) change nothing, nor do non-finite rows of other lists."""

    lengths, counts = [100, 64, 20], [2, 1, 1]
    cache, _, _ = filled(lengths, 2, 40, code, torch.bfloat16, capacity=256, device=DEV)
    q = torch.randn(4, 2, 40, device=DEV).bfloat16()
    seg, n = seg_of(counts, DEV), i32(lengths, DEV)
    want = ops.kv8_attention(q, cache, seg, n, 0.2)
    at = {w: D.code_positions(w, 5, torch.device(DEV)) for w in ("k", "v")}
    for l, length in enumerate(lengths):
        b = length // 64
        for which in ("k", "v"):
            codes, scale = getattr(cache, which + "_codes").view(torch.uint8), getattr(cache, which + "_scale")
            codes[l, :, b + 1 :] = 0x7F
            scale[l, :, b + 1 :] = math.nan
            flat = codes[l, :, b].reshape(2, -1)
            flat[:, at[which][length % 64 :]] = 0x7F
            codes[l, :, b] = flat.view(2, 5, 512)
            if length % 64 == 0:
                scale[l, :, b] = math.nan
    assert torch.equal(want, ops.kv8_attention(q, cache, seg, n, 0.2))
    cache.k_scale[1, :, 0] = math.nan                             # a list that holds a NaN: its own rows only
    got = ops.kv8_attention(q, cache, seg, n, 0.2)
    assert got[2].isnan().all() and torch.equal(got[[0, 1, 3]], want[[0, 1, 3]])


@pytest.mark.gpu
def test_attention_masks_inside_a_step_whose_later_rows_are_poisoned():
    """A block that only the later rows of a step reach may hold a NaN: the earlier row does not see it."""

    cache, _, _ = filled([65], 1, 16, torch.int8, torch.float32, capacity=128, device=DEV)
    cache.k_scale[0, 0, 1] = math.nan
    cache.v_scale[0, 0, 1] = math.nan
    q = torch.randn(2, 1, 16, device=DEV)
    got = ops.kv8_attention(q, cache, seg_of([2], DEV), i32([65], DEV), 0.2, max_rows=2)
    alone = ops.kv8_attention(q[:1], cache, seg_of([1], DEV), i32([64], DEV), 0.2)
    assert torch.equal(got[0], alone[0]) and got[1].isnan().all()


@pytest.mark.gpu
def test_attention_rows_behind_the_last_list_and_empty_steps():
    cache, _, _ = filled([100, 50], 2, 24, torch.int8, torch.float16, device=DEV)
    q = torch.randn(5, 2, 24, device=DEV).half()
    seg, n = seg_of([1, 1], DEV), i32([100, 50], DEV)
    got = ops.kv8_attention(q, cache, seg, n, 0.2)
    assert torch.equal(got[2:], torch.zeros_like(got[2:])) and got[:2].abs().sum() > 0
    out = torch.full((5, 2, 48), 3.0, dtype=torch.float16, device=DEV)[..., :24]        # a strided output
    ops.kv8_attention(q, cache, seg, n, 0.2, out=out)
    assert torch.equal(out[:2], got[:2]) and (out[2:] == 3.0).all()
    assert ops.kv8_attention(q[:0], cache, seg_of([0, 0], DEV), n, 0.2).shape == (0, 2, 24)
    none = ops.kv8_attention(q, cache, seg_of([0, 0], DEV), n, 0.2)
    assert torch.equal(none, torch.zeros_like(none))


@pytest.mark.gpu
def test_attention_with_more_lists_than_one_launch_holds():
    L = 4096 + 300
    counts = [1 if i % 7 == 0 or i >= 4090 else 0 for i in range(L)]
    lengths = [(i * 37) % 90 + 1 for i in range(L)]
    cache, _, _ = filled(lengths, 1, 16, torch.int8, torch.bfloat16, device=DEV)
    rows = sum(counts)
    q = torch.randn(rows + 1, 1, 16, device=DEV).bfloat16()
    seg = seg_of(counts, DEV)
    got = ops.kv8_attention(q, cache, seg, i32(lengths, DEV), 0.25)
    check_attention(q, cache, seg, lengths, 0.25, got)
    assert (got[rows] == 0).all()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    L, H, hd = 40, 16, 64
    cache = ops.kv8_cache(L, H, 110_016, hd, DEV)                 # 4.5 GB of codes for the keys, as much for the values
    assert cache.k_codes.numel() > 2 ** 32
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(140, H, hd, generator=g).bfloat16().to(DEV), torch.randn(140, H, hd, generator=g).bfloat16().to(DEV)
    counts = [0] * (L - 1) + [140]
    ops.kv8_append(cache, k, v, seg_of(counts, DEV), i32([0] * L, DEV), max_rows=140)
    ops.kv8_append(cache, k, v, seg_of(counts, DEV), i32([109_824] * L, DEV), max_rows=140)
    small = ops.kv8_cache(1, H, 192, hd, DEV)
    ops.kv8_append(small, k, v, seg_of([140], DEV), i32([0], DEV), max_rows=140)
    assert torch.equal(cache.k_codes[-1, :, :3], small.k_codes[0]) and torch.equal(cache.v_codes[-1, :, 1716:], small.v_codes[0])
    back = ops.kv8_read(cache, seg_of(counts, DEV), i32([109_824] * L, DEV), 140)
    assert torch.equal(back[1], ops.kv8_read(small, seg_of([140], DEV), i32([0], DEV), 140)[1])
    q = torch.randn(1, H, hd, generator=g).bfloat16().to(DEV)
    a = ops.kv8_attention(q, cache, seg_of([0] * (L - 1) + [1], DEV), i32([0] * (L - 1) + [140], DEV), 0.125)
    # (the two capacities divide the work differently, so the sums may differ in their last bits: both have the bound)
    check_attention(q, small, seg_of([1], DEV), [140], 0.125, a)
    check_attention(q, small, seg_of([1], DEV), [140], 0.125, ops.kv8_attention(q, small, seg_of([1], DEV), i32([140], DEV), 0.125))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_long_lines_are_shared_out_at_run_time(code):
    """Enough blocks that warps fetch units as they finish: the same values every time, rows that nothing cuts and rows
    that are cut many times."""

    g = torch.Generator(DEV).manual_seed(2)
    L, H, nb, U = 96, 4, 420, 2                                   # 161280 blocks, 63 for each of 2560 warps or fewer
    codes = [torch.randint(-127, 128, (L, H, nb, U, 512), generator=g, device=DEV, dtype=torch.int8) for _ in range(2)]
    if code != torch.int8:
        codes = [torch.where((c & 0x7F) == 0x7F, 0, c).view(code) for c in codes]    # (no NaN code: 0x7f and 0xff)
    scale = [torch.rand(L, H, nb, generator=g, device=DEV) * 0.02 for _ in range(2)]
    held = [torch.zeros(L, H, 2, 64, 16, device=DEV, dtype=torch.float16) for _ in range(2)]
    cache = D.KV8Cache(*codes, *scale, *held)
    lengths = [64 * nb - 17 * l if l % 8 else 60 + l for l in range(L)]
    q = torch.randn(L, H, 16, generator=g, device=DEV).half()
    seg, n = seg_of([1] * L, DEV), i32(lengths, DEV)
    runs = [ops.kv8_attention(q, cache, seg, n, 0.05) for _ in range(4)]
    assert all(torch.equal(runs[0], r) for r in runs)
    some = [0, 1, 8, 50, 95]
    part = D.KV8Cache(*(c.view(torch.int8)[some].view(code) for c in codes), *(t[some] for t in scale + held))
    check_attention(q[some], part, seg_of([1] * len(some)), [lengths[l] for l in some], 0.05, runs[0][some])


@pytest.mark.gpu
def test_first_calls_may_be_under_capture():
    cache, _, _ = filled([70, 20], 2, 72, torch.float8_e4m3fn, torch.float16, device=DEV)
    q = torch.randn(2, 2, 72, device=DEV).half()
    seg, n = seg_of([1, 1], DEV), i32([70, 20], DEV)
    wide = ops.kv8_cache(2, 2, 1 << 20, 104, DEV, torch.float8_e4m3fn, torch.float16)      # (units and a workspace)
    k, q2 = torch.randn(2, 2, 104, device=DEV).half(), torch.randn(2, 6, 104, device=DEV).half()
    p, x, d, u, w, lens = (t.to(DEV) for t in drafts(3, 2, 999, torch.float16, False, 5))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = ops.kv8_attention(q, cache, seg, n, 0.1)
        ops.kv8_append(wide, k, k, seg, n * 0)
        b = ops.kv8_attention(q2, wide, seg, n * 0 + 1, 0.1)
        c = ops.verify_draft(p, x, d, u, w, lens)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, ops.kv8_attention(q, cache, seg, n, 0.1))
    # one entry: its value, whatever the query
    back = ops.kv8_read(wide, seg, n * 0, 2, dtype=torch.float16)[1]
    assert torch.allclose(b.float(), back.repeat_interleave(3, 1).float(), rtol=2.0 ** -10)
    assert all(torch.equal(i, j) for i, j in zip(c, ops.verify_draft(p, x, d, u, w, lens)))


@pytest.mark.gpu
@pytest.mark.parametrize("capacity", [1024, 300_000])             # by tasks; by units with a workspace
def test_decode_step_in_graphs_and_on_streams(capacity):
    """Append and attention captured in two graphs that replay in turn, and on two streams at once."""

    def setup(seed):
        cache, _, _ = filled([700, 90, 33], 2, 40, torch.int8, torch.bfloat16, seed=seed, capacity=capacity, device=DEV)
        g = torch.Generator().manual_seed(seed)
        q, k, v = (torch.randn(3, 2, 40, generator=g).bfloat16().to(DEV) for _ in range(3))
        return cache, q, k, v, seg_of([1, 1, 1], DEV), i32([700, 90, 33], DEV)

    def step(cache, q, k, v, seg, start):
        ops.kv8_append(cache, k, v, seg, start)
        return ops.kv8_attention(q, cache, seg, start + 1, 0.1)

    sets = [setup(i) for i in range(2)]
    want = [step(*s) for s in sets]
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*s))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(want[i], x) for i in range(2) for x in got[i])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("V", [1, 5, 1000, 4097, 50257, 100263, 700001])
def test_verification_kernel(kind, V):
    for n, greedy in ((0, False), (4, False), (3, True), (40, False)):
        if n == 40 and V > 5000:
            continue
        p, x, q, u, w, lens = drafts(9, n, V, kind, greedy, n + V)
        for use in (lens, None):
            want = ops.verify_draft(p, x, q, u, w, use)
            d = lambda t: None if t is None else t.to(DEV)          # noqa: E731
            got = ops.verify_draft(d(p), d(x), d(q), d(u), d(w), d(use))
            assert torch.equal(want[0], got[0].cpu()) and torch.equal(want[1], got[1].cpu()), (n, greedy)
            wide = torch.full((9, n + 3, V + 5), math.nan, dtype=kind, device=DEV)          # rows inside a padded buffer
            wide[:, 1 : n + 2, 3 : V + 3] = d(p)
            got = ops.verify_draft(wide[:, 1 : n + 2, 3 : V + 3], d(x).int(), d(q), d(u), d(w), d(use))
            assert torch.equal(want[0], got[0].cpu()) and torch.equal(want[1], got[1].cpu()), (n, greedy)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_verification_kernel_on_many_sequences(kind):
    for B, n, V, greedy in ((300, 2, 5003, False), (90, 3, 50257, False), (700, 1, 130, True)):
        p, x, q, u, w, lens = drafts(B, n, V, kind, greedy, B)
        want = ops.verify_draft(p, x, q, u, w, lens)
        d = lambda t: None if t is None else t.to(DEV)              # noqa: E731
        got = ops.verify_draft(d(p), d(x), d(q), d(u), d(w), d(lens))
        assert torch.equal(want[0], got[0].cpu()) and torch.equal(want[1], got[1].cpu())


@pytest.mark.gpu
def test_borders_of_verification_kernel():
    for p, x, q, u, w, accepted, token in edge_cases():
        d = lambda t: None if t is None else t.to(DEV)              # noqa: E731
        a, t = ops.verify_draft(d(p), d(x), d(q), d(u), d(w))
        assert (a.tolist(), t.tolist()) == ([accepted], [token])
