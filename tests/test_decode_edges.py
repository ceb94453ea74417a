"""The decoding ops and decode states at the edges: waits that run out, row bounds, threads, other callers' decode states."""

import math

import pytest
import torch

from nestor_b200 import ops
from nestor_b200.ops import decode as D
from test_decode_ops import CODES, TYPES, check_attention, filled, same, to, values64

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
@pytest.mark.parametrize("code", CODES)
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


@pytest.mark.gpu
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("capacity", [64, 300_000])               # by tasks; by units with a workspace
def test_rows_before_the_first_list_are_zeros_and_reported(capacity, given):
    from nestor_b200.ops import _lib
    dev = torch.device(DEV, 0)
    cache, _, _ = filled([3, 50], 2, 24, torch.int8, torch.bfloat16, capacity=capacity, device=DEV)
    q = torch.randn(7, 2, 24, device=DEV).bfloat16()
    n = i32([3, 50], DEV)
    want = ops.kv8_attention(q[2:], cache, seg_of([1, 2], DEV), n, 0.2, max_rows=2)
    _lib.check_status(dev)
    held = [torch.full_like(q, math.nan) for _ in range(8)]       # (what an allocation of this size finds)
    out = torch.full_like(q, 3.0) if given else None
    del held
    got = ops.kv8_attention(q, cache, i32([2, 3, 5], DEV), n, 0.2, max_rows=2, out=out)
    with pytest.raises(RuntimeError, match="row bounds"):
        _lib.check_status(dev)
    assert (got[:2] == 0).all() and torch.equal(got[2:5], want[:3]) and (got[5:] == (3 if given else 0)).all()


@pytest.mark.gpu
def test_rows_before_the_first_list_cost_no_other_row():
    """Append drops them and read gives zeros for them, both report them, and the rows behind them are served."""

    from nestor_b200.ops import _lib
    dev = torch.device(DEV, 0)
    a, b = (ops.kv8_cache(3, 2, 128, 24, DEV) for _ in range(2))
    k, v = (torch.randn(9, 2, 24, device=DEV).bfloat16() for _ in range(2))
    zero = i32([0, 0, 0], DEV)
    ops.kv8_append(a, k[2:], v[2:], i32([0, 1, 1, 5], DEV), zero, max_rows=64)
    want = ops.kv8_read(a, i32([0, 1, 1, 5], DEV), zero, 6, max_rows=64)
    _lib.check_status(dev)
    ops.kv8_append(b, k, v, i32([2, 3, 3, 7], DEV), zero, max_rows=64)
    with pytest.raises(RuntimeError, match="row bounds"):
        _lib.check_status(dev)
    assert same(a, b)
    got = ops.kv8_read(b, i32([2, 3, 3, 7], DEV), zero, 8, max_rows=64)
    with pytest.raises(RuntimeError, match="row bounds"):
        _lib.check_status(dev)
    for x, y in zip(want, got):
        assert (y[:2] == 0).all() and torch.equal(x, y[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("capacity", [1024, 20_032])              # the same entries by tasks and by units
def test_small_weights_beside_a_dominating_one(code, kind, capacity):
    """One entry 20 above all others, with the value zero: what is left are the others, each with e^-20 of its weight.

    With ``m = sum_i p_i |v_i|``: scores and exponentials as in ``attention64``, whose relative error ``e`` of a weight
    moves the output by at most ``2 e m`` here (all terms are kept, not bounded by the largest value); the weights, two
    fp16 numbers, 2^-21 of themselves and 2^-40 of their block's largest one, which is theirs but for the first block; for
    bf16, one number, 2^-11 of themselves and 2^-32 of the largest; the fp32 sums of products of one sign
    ``(n / 16 + 16) 2^-23 m``. int8 codes with 16-bit queries enter as 128 more: the four to eight products of a block and the
    removal of the 128 round sums of up to 128 times the block's weights, ``10 2^-23 128 sum(p)`` in all. The output is
    rounded by half a step, which for outputs below the type's smallest normal number ``t`` (2^-14 in fp16; 1e-6 is below
    it) is that of ``t``: ``t eps / 2`` = 2^-25.
    """

    n, hd = min(capacity, 20_001), 8
    cache = ops.kv8_cache(1, 1, capacity, hd, DEV, code, torch.float32)
    g = torch.Generator().manual_seed(4)
    k = torch.zeros(n, 1, hd)
    k[0, 0, 0] = 1
    v = torch.rand(n, 1, hd, generator=g) * 0.5 + 0.5
    v[0] = 0
    ops.kv8_append(cache, k.to(DEV), v.to(DEV), seg_of([n], DEV), i32([0], DEV), max_rows=n)
    q = torch.zeros(2, 1, hd)
    q[0, 0, 0], q[1, 0, 0] = 20, 10
    q = q.to(kind)
    got = ops.kv8_attention(q.to(DEV), cache, seg_of([2], DEV), i32([n], DEV), 1.0, max_rows=2).double().cpu()
    host = to(cache, "cpu")
    for a in range(2):
        see = n - 1 + a
        kk, vv = (values64(host, w, 0, n)[0, :see] for w in ("k", "v"))
        s = kk @ q[a, 0].double()
        p = torch.softmax(s, 0)
        want, m = p @ vv, p @ vv.abs()
        lift = 128 if kind != torch.float32 and code == torch.int8 else 0
        big = float(s.abs().max()) + lift * float(host.k_scale.max()) * float(q[a].abs().sum())
        e = math.expm1(2 * (big * (hd + 8) * 2.0 ** -23 + 2.0 ** -22 + 2 * float(s.abs().max()) * 1.45 * 2.0 ** -23))
        e += 2.0 ** -11 if kind == torch.bfloat16 else 2.0 ** -21
        grain = n * 2.0 ** -32 if kind == torch.bfloat16 else 64 * 2.0 ** -40
        sums = (see / 16 + 16) * 2.0 ** -23 * m + (10 * 2.0 ** -23 * 128 * float(host.v_scale.max()) if lift else 0.0)
        tol = 2 * e * m + sums + grain + torch.finfo(kind).eps / 2 * (want.abs() * 1.01).clamp_min(torch.finfo(kind).tiny)
        off = (got[a, 0] - want).abs()
        assert (off <= tol).all(), (a, float((off / tol).max()), float((off / want).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("code", CODES)
def test_queries_of_a_wide_range(code, kind):
    """A large element where the keys are zero, and elements 2^-18 of it that decide against keys 2^12 times larger."""

    n, hd = 90, 40
    g = torch.Generator().manual_seed(6)
    k = torch.randn(n, 1, hd, generator=g) * 2.0 ** 12
    k[:, :, 3] = 0
    v = torch.randn(n, 1, hd, generator=g)
    cache = ops.kv8_cache(1, 1, 128, hd, DEV, code, torch.float32)
    ops.kv8_append(cache, k.to(DEV), v.to(DEV), seg_of([n], DEV), i32([0], DEV), max_rows=n)
    q = torch.randn(3, 1, hd, generator=g) * 2.0 ** -9
    q[:, :, 3] = 2.0 ** 9 * 1.25
    q = q.to(kind)
    seg = seg_of([3], DEV)
    got = ops.kv8_attention(q.to(DEV), cache, seg, i32([n], DEV), 0.25, max_rows=3)
    host = to(cache, "cpu")
    kk = values64(host, "k", 0, n)[0]
    # (the bound without the zero keys' dimension: what stands there adds nothing to any score, but int8 codes carry it
    # with a factor of 128, which is part of the bound)
    assert float((kk @ q[0, 0].double()).abs().max()) > 8
    check_attention(q, cache, seg, [n], 0.25, got)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("top", [2.0 ** 100, 2.0 ** 124, 3.38e38])
def test_queries_near_the_end_of_their_range(code, kind, top):
    """Scores that differ by far more than the exponential can hold: the best entry's value (one weight, an exact sum),
    rounded by half a step of the output's type."""

    n, hd = 70, 8
    g = torch.Generator().manual_seed(2)
    k = torch.rand(n, 1, hd, generator=g) * 0.01
    k[61, 0, 2] = 0.02
    v = torch.randn(n, 1, hd, generator=g)
    cache = ops.kv8_cache(1, 1, 128, hd, DEV, code, torch.float32)
    ops.kv8_append(cache, k.to(DEV), v.to(DEV), seg_of([n], DEV), i32([0], DEV), max_rows=n)
    q = torch.zeros(1, 1, hd)
    q[0, 0, 2] = top
    got = ops.kv8_attention(q.to(kind).to(DEV), cache, seg_of([1], DEV), i32([n], DEV), 1.0)[0, 0].double().cpu()
    want = values64(to(cache, "cpu"), "v", 0, n)[0, 61]
    assert ((got - want).abs() <= torch.finfo(kind).eps / 2 * want.abs() * 1.01 + 2.0 ** -20).all()


class OnDevice:
    """What ``use_kernels`` looks at."""

    is_cuda = True


def test_regions_of_two_threads_do_not_mix():
    """Two threads that decode at once enter and leave their regions in any order: each sees its own, and none is left."""

    import threading
    turn, seen, failed = [threading.Event() for _ in range(6)], {}, []

    def wait(i):
        if not turn[i].wait(20):
            failed.append(i)

    def a():
        with ops.oracle_ops():
            turn[0].set()
            wait(1)                                               # b is in its region
            with ops.kernel_ops(True):
                turn[2].set()
                seen["a"] = ops.use_kernels(OnDevice)
                wait(3)                                           # b has left its region
            seen["a behind"] = ops.use_kernels(OnDevice)
        turn[4].set()

    def b():
        wait(0)
        with ops.oracle_ops():
            turn[1].set()
            wait(2)                                               # a is in both
            seen["b"] = ops.use_kernels(OnDevice)
        turn[3].set()
        wait(4)
        seen["b behind"] = ops.use_kernels(OnDevice)

    threads = [threading.Thread(target=f) for f in (a, b)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    assert seen == {"a": True, "a behind": False, "b": False, "b behind": True}
    assert ops.use_kernels(OnDevice)


def test_nested_regions():
    at = lambda: ops.use_kernels(OnDevice)                        # noqa: E731
    with ops.oracle_ops():
        assert not at()
        inner = ops.kernel_ops(True)
        with inner:
            assert at()
            with ops.oracle_ops():
                assert not at()
                with inner:
                    assert at()
                assert not at()
            assert at()
        with ops.kernel_ops(False):
            assert not at()
        assert not at()
    assert at()
    with pytest.raises(KeyError):
        with ops.oracle_ops(), ops.kernel_ops(True):
            raise KeyError
    assert at()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_keywords_in_any_order(device):
    cache = ops.kv8_cache(2, 2, 64, 8, device)
    rows = torch.randn(2, 2, 8, device=device).bfloat16()
    seg, zero, one = (i32(x, device) for x in ([0, 1, 2], [0, 0], [1, 1]))
    ops.kv8_append(max_rows=1, start=zero, seg_start=seg, v=rows, k=rows, cache=cache)
    ops.kv8_truncate(lengths=one, cache=cache)
    back = ops.kv8_read(rows=2, start=zero, seg_start=seg, cache=cache)[1]
    got = ops.kv8_attention(scale=0.5, max_rows=1, lengths=one, seg_start=seg, cache=cache, q=rows)
    assert torch.equal(got, ops.kv8_attention(rows, cache, seg, one, 0.5))
    assert torch.allclose(got.float(), back, rtol=2.0 ** -8)      # one entry: its value
    p = torch.softmax(torch.randn(2, 3, 9, device=device), -1)
    x, u, w = torch.zeros(2, 2, dtype=torch.int32, device=device), torch.rand(2, 2, device=device), torch.rand(2, device=device)
    a = ops.verify_draft(draft_probs=None, sample_u=w, accept_u=u, draft_tokens=x, target_probs=p)
    assert all(torch.equal(i, j) for i, j in zip(a, ops.verify_draft(p, x, None, u, w)))


def test_calls_without_their_first_argument():
    cache = ops.kv8_cache(1, 1, 64, 8)
    for call in (lambda: ops.kv8_truncate(), lambda: ops.kv8_truncate(lengths=i32([1])), lambda: ops.kv8_attention(cache=cache, scale=1.0)):
        with pytest.raises(TypeError, match="argument"):
            call()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_dual_tensors_are_refused(device):
    """Forward-mode derivatives would be lost without a word, under no_grad too."""

    import torch.autograd.forward_ad as fwd
    cache = ops.kv8_cache(1, 1, 64, 8, device, open_dtype=torch.float32)
    rows, seg, n = torch.randn(1, 1, 8, device=device), i32([0, 1], device), i32([0], device)
    p = torch.full((1, 2, 4), 0.25, device=device)
    x, u, w = torch.zeros(1, 1, dtype=torch.int32, device=device), torch.rand(1, 1, device=device), torch.rand(1, device=device)
    with torch.no_grad(), fwd.dual_level():
        dual, dual_p = fwd.make_dual(rows, rows), fwd.make_dual(p, p)
        for call in (lambda: ops.kv8_append(cache, dual, rows, seg, n), lambda: ops.kv8_append(cache, rows, dual, seg, n),
                     lambda: ops.kv8_attention(dual, cache, seg, n, 1.0), lambda: ops.kv8_attention(rows, cache, seg, n, 1.0, out=dual),
                     lambda: ops.verify_draft(dual_p, x, None, u, w), lambda: ops.verify_draft(p, x, dual_p[:, :1], u, w)):
            with pytest.raises(RuntimeError, match="dual tensors"):
                call()
        ops.kv8_append(cache, rows, rows, seg, n)                # (others are welcome inside such a level)
        ops.kv8_attention(rows, cache, seg, n + 1, 1.0)
        ops.verify_draft(p, x, p[:, :1], u, w)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: ops.kv8_attention(q, cache, seg, n + 1, 1.0), (rows,), (rows,))


class SumState:
    """A decode state of another backbone, with the one attribute that stepwise decoding has always asked for."""

    def __init__(self, B, width, device):
        self.length, self.sum = 0, torch.zeros(B, width, device=device)


class SumBackbone(torch.nn.Module):
    def init_kv_cache(self, batch_size, max_len, device, dtype=torch.float32):
        assert dtype == torch.float32
        return SumState(batch_size, 128, device)

    def forward_step(self, x0, pos, cache, cd):
        assert pos.tolist() == [cache.length] * x0.shape[0] and pos.dtype == torch.long
        cache.sum = 0.7 * cache.sum + x0 * (1 + pos[0])
        cache.length += 1
        return cache.sum.to(cd), {}


def test_another_backbones_decode_state(tiny_scale):
    from test_decode_8bit import tiny
    m = tiny(tiny_scale, "dense", 2)
    m.backbone = SumBackbone()
    ids = torch.randint(0, 100263, (2, 6))
    x = m.adapter(ids)
    with torch.no_grad():
        state, want = torch.zeros(2, x.shape[-1]), []
        for t in range(6):
            state = 0.7 * state + x[:, t] * (1 + t)
            want.append(m.head(state, torch.float32).float())
    cache = m.init_kv_cache(2, 6)
    for t in range(3):
        assert torch.equal(m.decode_step(ids[:, t], cache), want[t])
    assert torch.equal(m.decode_step(ids[:, 3:], cache), torch.stack(want[3:], 1))       # several tokens: step by step
    out = m.generate(ids, 4)
    assert out.shape == (2, 10) and torch.equal(out[:, :6], ids) and torch.equal(out[:, 6], want[5].argmax(-1))
    with pytest.raises(ValueError, match="SumBackbone does not offer"):
        m.generate(ids, 4, draft=m)


def test_an_fp32_state_steps_its_first_sequences(tiny_scale):
    """A state made for four sequences decodes two of them, then all: positions count steps, as they always did, and
    taking tokens back touches the sequences that were fed."""

    from test_decode_8bit import tiny
    m = tiny(tiny_scale, "nestor", 4)
    ids = torch.randint(0, 100263, (4, 9))
    two, four = m.init_kv_cache(2, 12), m.init_kv_cache(4, 12)
    for t in range(4):
        assert torch.equal(m.decode_step(ids[:2, t], two), m.decode_step(ids[:2, t], four))
    assert four.length == 4 and four.positions.tolist() == [4] * 4
    alone = m.init_kv_cache(4, 12)
    for t in range(4):
        m.decode_step(ids[:, t], alone)
    for blk in alone.blocks:
        for layer in blk:
            layer.count[2:] = 0                                   # (what the two that were not fed hold: nothing)
    assert torch.allclose(m.decode_step(ids[:, 4], four), m.decode_step(ids[:, 4], alone), atol=1e-5)
    four.rollback(torch.tensor([2, 1, 1, 0]))                     # (one step is all that the last two can give back)
    assert four.positions.tolist() == [3, 4, 4, 5]
    four.rollback(torch.tensor([0, 0, 0, 1]))
    with pytest.raises(ValueError, match="taken back"):
        four.rollback(torch.tensor([0, 0, 0, 1]))
    with torch.no_grad():
        full = m(ids[:2]).pred.float()
    step = m.decode_step(torch.stack([ids[0, 3], ids[1, 4], ids[2, 4], ids[3, 4]]), four)
    assert torch.allclose(step[0], full[0, 3], atol=2e-4, rtol=1e-4) and torch.allclose(step[1], full[1, 4], atol=2e-4, rtol=1e-4)
    for state in (two, m.init_kv_cache(2, 8, dtype=torch.int8)):
        with pytest.raises(ValueError, match="tokens for 3"):
            m.decode_step(ids[:3, 0], state)
    with pytest.raises(ValueError, match="tokens for 1"):
        m.decode_step(ids[:1, 0], m.init_kv_cache(2, 8, dtype=torch.int8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.int8])
def test_a_decode_state_is_reset_by_its_counts_and_length(dtype, tiny_scale):
    from test_decode_8bit import tiny
    m = tiny(tiny_scale, "nestor", 5)
    ids = torch.randint(0, 100263, (2, 5))
    cache = m.init_kv_cache(2, 6, dtype=dtype)
    first = [m.decode_step(ids[:, t], cache) for t in range(5)]
    for blk in cache.blocks:
        for layer in blk:
            layer.count.zero_()
    cache.length = 0
    assert cache.positions.tolist() == [0, 0]
    with pytest.raises(ValueError, match="taken back"):
        cache.rollback(torch.tensor([1, 1]))
    assert all(torch.equal(first[t], m.decode_step(ids[:, t], cache)) for t in range(5))
    assert cache.length == 5


@pytest.mark.parametrize("S", [37, 33, 16, 1])
def test_a_prompt_asks_the_head_for_its_last_row(S, tiny_scale, monkeypatch):
    from test_decode_8bit import tiny
    m = tiny(tiny_scale, "nestor", 6)
    monkeypatch.setattr(m, "PREFILL", 16)
    prompt = torch.randint(0, 100263, (2, S))
    asked, head = [], m.head.forward
    monkeypatch.setattr(m.head, "forward", lambda h, *a, **kw: (asked.append(h.shape[0]), head(h, *a, **kw))[1])
    with torch.no_grad():
        got = m._prefill(prompt, m.init_kv_cache(2, 40, dtype=torch.int8))
    assert asked == [2] and m._prefill(prompt[:, :0], m.init_kv_cache(2, 4, dtype=torch.int8)) is None
    cache = m.init_kv_cache(2, 40, dtype=torch.int8)
    for a in range(0, S, 16):
        want = m.decode_step(prompt[:, a : a + 16], cache)
    assert torch.allclose(got, want if want.dim() == 2 else want[:, -1], atol=1e-5)
    out = m.generate(prompt, 2, cache_dtype=torch.int8)
    assert torch.equal(out[:, S], got.argmax(-1))


def test_a_refused_or_failing_generation_leaves_the_training_mode(tiny_scale, monkeypatch):
    from test_decode_8bit import tiny
    m, draft = tiny(tiny_scale, "moe", 5).train(), tiny(tiny_scale, "dense", 6).train()
    prompt = torch.randint(0, 100263, (2, 4))
    with pytest.raises(ValueError, match="draft_tokens"):
        m.generate(prompt, 4, draft=draft, draft_tokens=0)
    with torch.no_grad():
        m.head.weight.fill_(float("nan"))
    with pytest.raises(RuntimeError, match="no token to draw"):
        m.generate(prompt, 4, 0.8, torch.Generator().manual_seed(0), torch.int8, draft, 3)
    assert m.training and draft.training and all(x.training for x in m.modules()) and all(x.training for x in draft.modules())
    monkeypatch.setattr(m, "decode_step", lambda *a, **kw: 1 / 0)
    with pytest.raises(ZeroDivisionError):
        m.generate(prompt, 4)
    assert m.training
    draft.eval()
    draft.generate(prompt, 2)
    assert not draft.training


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [False, True])
def test_generation_reports_what_its_kernels_report(drafted, tiny_scale, monkeypatch):
    """A wait that ran out leaves NaN logits: an error before anything is drawn from them, and the device goes on."""

    from nestor_b200.ops import _lib, cuda_decode
    from test_decode_8bit import tiny
    m = tiny(tiny_scale, "nestor", 8).cuda()
    kw = dict(draft=tiny(tiny_scale, "dense", 9).cuda(), draft_tokens=3) if drafted else {}
    prompt = torch.randint(0, 100263, (3, 9), device=DEV)
    g = torch.Generator(DEV)
    want = m.generate(prompt, 5, 0.7, g.manual_seed(1), torch.int8, **kw)
    monkeypatch.setattr(cuda_decode, "WAIT_POLLS", 0)
    with pytest.raises(RuntimeError, match="wait gave up"):
        m.generate(prompt, 5, 0.7, g.manual_seed(1), torch.int8, **kw)
    monkeypatch.undo()
    assert torch.equal(want, m.generate(prompt, 5, 0.7, g.manual_seed(1), torch.int8, **kw))
    _lib.status_word(torch.device(DEV, 0)).fill_(7)
    with pytest.raises(RuntimeError, match="capacity"):
        m.generate(prompt, 1, 0.0, None, torch.int8, **kw)
    assert torch.isfinite(m.generate(prompt, 2)).all()            # an fp32 state runs no kernel that could report
    _lib.check_status(torch.device(DEV, 0))


def test_generation_on_the_cpu_asks_no_device(tiny_scale, monkeypatch):
    from nestor_b200.ops import _lib
    from test_decode_8bit import tiny
    monkeypatch.setattr(_lib, "check_status", lambda device: 1 / 0)
    m = tiny(tiny_scale, "dense", 5)
    assert not m.init_kv_cache(1, 4, dtype=torch.int8).kernels
    assert m.generate(torch.randint(0, 100263, (1, 3)), 2, cache_dtype=torch.int8).shape == (1, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd", [30, 40, 101])
def test_long_appends_that_begin_inside_a_block(code, kind, hd):
    """Pieces of a prompt: a list begins anywhere in a block and goes on over two further blocks and more. The originals
    that were kept show when the list steps back and goes on."""

    g = torch.Generator().manual_seed(hd)
    L, H = 7, 2
    host = ops.kv8_cache(L, H, 900, hd, "cpu", code, kind)
    dev = to(host, DEV)
    at = [0] * L
    rounds = [([10, 63, 1, 64, 65, 33, 0], 0), ([130, 200, 193, 120, 191, 95, 129], 0), ([300, 1, 128, 129, 0, 160, 64], 0),
              ([1, 2, 64, 1, 70, 3, 5], 33), ([140, 150, 1, 190, 260, 64, 130], 64), ([0] * L, 50)]
    for i, (counts, back) in enumerate(rounds):
        if back:
            at = [max(0, a - back) for a in at]
            ops.kv8_truncate(host, i32(at))
            ops.kv8_truncate(dev, i32(at, DEV))
            assert same(host, dev), i
        rows = sum(counts) + 1
        k, v = (torch.randn(rows, H, hd, generator=g).to(kind) * (1 + torch.arange(rows) % 5).view(-1, 1, 1)).to(kind), torch.randn(rows, H, hd, generator=g).to(kind)
        for cache, d in ((host, "cpu"), (dev, DEV)):
            ops.kv8_append(cache, k.to(d), v.to(d), seg_of(counts, d), i32(at, d), max_rows=max(1, *counts))
        assert same(host, dev), i
        at = [a + n for a, n in zip(at, counts)]
    from nestor_b200.ops import _lib
    _lib.check_status(torch.device(DEV, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("kind,hd,group", [(torch.bfloat16, 40, 1), (torch.float32, 60, 1), (torch.float16, 80, 2)])
def test_a_prompt_in_pieces(code, kind, hd, group):
    """Appended and attended to in pieces, as a model feeds a prompt: many rows a list, lists that begin inside blocks."""

    g = torch.Generator().manual_seed(hd)
    L, H = 3, 2
    cache = ops.kv8_cache(L, H, 600, hd, DEV, code, kind)
    at = [0] * L
    for counts in ([170, 91, 33], [150, 0, 131], [70, 193, 1]):
        seg, rows = seg_of(counts, DEV), sum(counts)
        k, v = (torch.randn(rows, H, hd, generator=g).to(kind).to(DEV) for _ in range(2))
        ops.kv8_append(cache, k, v, seg, i32(at, DEV), max_rows=max(counts))
        at = [a + n for a, n in zip(at, counts)]
        q = (torch.randn(rows, H * group, hd, generator=g) * 2).to(kind).to(DEV)
        got = ops.kv8_attention(q, cache, seg, i32(at, DEV), 1 / hd ** 0.5, max_rows=max(counts))
        check_attention(q, cache, seg, at, 1 / hd ** 0.5, got)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hd,group", [(30, 3), (64, 1), (64, 4), (80, 2), (101, 1), (128, 8)])
def test_attention_in_pieces_that_are_joined(code, kind, hd, group):
    """Units and the join with every width class, one and two column tiles and several tiles a list."""

    lengths, counts = [3000, 130, 700, 1], [5, 3, 1, 1]
    cache, _, _ = filled(lengths, 2, hd, code, kind, seed=hd, capacity=8256, device=DEV)
    g = torch.Generator().manual_seed(8)
    q = (torch.randn(10, 2 * group, hd, generator=g) * torch.randn(10, 2 * group, 1, generator=g).exp() * 2).to(kind).to(DEV)
    seg = seg_of(counts, DEV)
    got = ops.kv8_attention(q, cache, seg, i32(lengths, DEV), 1 / hd ** 0.5, max_rows=5)
    check_attention(q, cache, seg, lengths, 1 / hd ** 0.5, got)
    assert torch.equal(got, ops.kv8_attention(q, cache, seg, i32(lengths, DEV), 1 / hd ** 0.5, max_rows=5))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("code", CODES)
def test_long_lines_of_wide_heads(code, kind):
    """Units fetched at run time with the ring of half blocks, two column tiles, several tiles a list."""

    L, H, blocks, hd, group = 24, 4, 420, 104, 4
    cache = random_cache(L, H, blocks, hd, code, 5, kind)
    counts, lengths = [5] * L, [blocks * 64 - 17 * l if l % 8 else 60 + l for l in range(L)]
    g = torch.Generator().manual_seed(9)
    q = torch.randn(5 * L, H * group, hd, generator=g).to(kind).to(DEV)
    got = ops.kv8_attention(q, cache, seg_of(counts, DEV), i32(lengths, DEV), 0.05, max_rows=5)
    for l in (1, 8, 23):
        part = D.KV8Cache(*(c.view(torch.int8)[l : l + 1].view(code) for c in (cache.k_codes, cache.v_codes)),
                          *(t[l : l + 1] for t in (cache.k_scale, cache.v_scale, cache.k_open, cache.v_open)))
        check_attention(q[5 * l : 5 * l + 5], part, seg_of([5], DEV), [lengths[l]], 0.05, got[5 * l : 5 * l + 5])
    assert torch.equal(got, ops.kv8_attention(q, cache, seg_of(counts, DEV), i32(lengths, DEV), 0.05, max_rows=5))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_the_join_of_many_items(code):
    """More (row, head) items than 32 for each multiprocessor, lists of one to seven blocks that units cut anywhere."""

    L = 400
    lengths = [1 + (l * 61) % 440 for l in range(L)]
    cache, _, _ = filled(lengths, 16, 24, code, torch.bfloat16, seed=3, device=DEV)
    q = torch.randn(L, 16, 24, device=DEV).bfloat16()
    assert L * 16 > 32 * torch.cuda.get_device_properties(0).multi_processor_count
    seg = seg_of([1] * L, DEV)
    got = ops.kv8_attention(q, cache, seg, i32(lengths, DEV), 0.2)
    check_attention(q, cache, seg, lengths, 0.2, got)


@pytest.mark.gpu
def test_greedy_decoding_with_drafts_on_the_gpu_is_the_models_own(tiny_scale):
    """Over an fp32 state the scoring of a round is the same single steps, so the tokens are the same."""

    from test_decode_8bit import tiny
    m, other = tiny(tiny_scale, "nestor", 3).cuda(), tiny(tiny_scale, "dense", 4).cuda()
    near = tiny(tiny_scale, "nestor", 3).cuda()
    torch.manual_seed(11)
    with torch.no_grad():
        for p in near.parameters():
            p.add_(torch.randn_like(p) * p.abs().mean() * 0.02)
    prompt = torch.randint(0, 100263, (3, 5), device=DEV)
    want = m.generate(prompt, 12)
    for draft, n in ((m, 4), (other, 1), (near, 3), (near, 6)):
        assert torch.equal(want, m.generate(prompt, 12, draft=draft, draft_tokens=n))


@pytest.mark.gpu
def test_a_cache_of_given_tensors_brings_the_status_word(monkeypatch):
    """Not its first step, which may be under capture: the word would live in that graph's memory."""

    from nestor_b200.ops import _lib
    cache = ops.kv8_cache(1, 1, 64, 8, DEV)
    monkeypatch.setattr(_lib, "_status", {})
    D.KV8Cache(*(getattr(cache, f) for f in ("k_codes", "v_codes", "k_scale", "v_scale", "k_open", "v_open")))
    assert list(_lib._status) == [0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.int8])
def test_a_decode_step_leaves_other_threads_ops_alone(dtype, tiny_scale, monkeypatch):
    import threading
    from nestor_b200.models.nestor import Layer
    from test_decode_8bit import tiny
    m = tiny(tiny_scale, "nestor", 5)
    seen, step = [], Layer.attention_step

    def look(self, *args):
        t = threading.Thread(target=lambda: seen.append(ops.use_kernels(OnDevice)))
        t.start()
        t.join()
        seen.append(ops.use_kernels(OnDevice))
        return step(self, *args)

    monkeypatch.setattr(Layer, "attention_step", look)
    m.decode_step(torch.randint(0, 100263, (2,)), m.init_kv_cache(2, 4, dtype=dtype))
    assert seen and all(seen[::2]) and not any(seen[1::2])
