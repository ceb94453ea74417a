"""Stepwise decoding over the 8-bit cache, steps of several tokens, taking tokens back, and decoding with drafts."""

import dataclasses as dc

import pytest
import torch

from nestor_b200 import ops


class ExactCache:
    """Stands in for the 8-bit ops with the same interface and full-precision storage, so that what is tested is how the
    model packs, appends, attends and takes back."""

    def __init__(self, monkeypatch):
        self.held = {}
        for name in ("kv8_append", "kv8_attention", "kv8_truncate"):
            monkeypatch.setattr(ops, name, getattr(self, name))

    def of(self, cache):
        if id(cache) not in self.held:
            L, H, n, D = cache.lists, cache.heads, cache.capacity, cache.head_dim
            self.held[id(cache)] = (cache, torch.zeros(L, n, H, D), torch.zeros(L, n, H, D))
        return self.held[id(cache)][1:]

    def kv8_append(self, cache, k, v, seg_start, start, max_rows=1):
        seg, at = seg_start.tolist(), start.tolist()
        for l, s in enumerate(at):
            n = seg[l + 1] - seg[l]
            assert n <= max_rows and s + n <= cache.capacity
            for mine, new in zip(self.of(cache), (k, v)):
                mine[l, s : s + n] = new[seg[l] : seg[l + 1]]

    def kv8_attention(self, q, cache, seg_start, lengths, scale, max_rows=1, out=None):
        seg, size = seg_start.tolist(), lengths.tolist()
        out = torch.zeros_like(q)
        keys, values = self.of(cache)
        for l, length in enumerate(size):
            n = seg[l + 1] - seg[l]
            for a in range(n):
                see = length - (n - 1 - a)
                p = torch.softmax(torch.einsum("hd,ehd->he", q[seg[l] + a], keys[l, :see]) * scale, -1)
                out[seg[l] + a] = torch.einsum("he,ehd->hd", p, values[l, :see])
        return out

    def kv8_truncate(self, cache, lengths):
        for l, n in enumerate(lengths.tolist()):
            for mine in self.of(cache):
                mine[l, n:] = float("nan")          # nothing may look behind a list's end


def tiny(scale, family, seed=0, **backbone):
    from nestor_b200.models import Model
    torch.manual_seed(seed)
    cfg = scale.build_experiment(family, "tiny").jobs[0].model
    cfg = dc.replace(cfg, backbone_config=dc.replace(cfg.backbone_config, **backbone)) if backbone else cfg
    m = Model.from_config(cfg).eval()
    with torch.no_grad():
        for n, p in m.named_parameters():          # make the depth reads non-trivial
            if "query" in n:
                p.normal_(0, 0.5)
            if "value_gains" in n:
                p.uniform_(0.5, 1.5)
    return m


@pytest.mark.parametrize("family", ["nestor", "moe", "dense"])
def test_steps_of_several_tokens_match_the_full_forward(family, tiny_scale, monkeypatch):
    ExactCache(monkeypatch)
    m = tiny(tiny_scale, family)
    ids = torch.randint(0, 100263, (2, 24))
    with torch.no_grad():
        full = m(ids).pred.float()
    cache = m.init_kv_cache(2, 24, dtype=torch.int8)
    at = 0
    for n in (7, 1, 11, 5):
        step = m.decode_step(ids[:, at : at + n] if n > 1 else ids[:, at], cache)
        step = step if n > 1 else step.unsqueeze(1)
        assert torch.allclose(step, full[:, at : at + n], atol=2e-4, rtol=1e-4)
        at += n
    assert cache.length == 24 and cache.positions.tolist() == [24, 24]
    with pytest.raises(ValueError, match="cache"):
        m.decode_step(ids[:, :1], cache)
    with pytest.raises(ValueError, match="tokens for 4"):
        m.decode_step(torch.cat((ids, ids))[:, 0], m.init_kv_cache(2, 8, dtype=torch.int8))


@pytest.mark.parametrize("eight_bit", [True, False])
def test_tokens_are_taken_back_sequence_by_sequence(eight_bit, tiny_scale, monkeypatch):
    ExactCache(monkeypatch)
    m = tiny(tiny_scale, "nestor", 1)
    ids = torch.randint(0, 100263, (3, 20))
    with torch.no_grad():
        full = m(ids).pred.float()
    cache = m.init_kv_cache(3, 40, dtype=torch.int8 if eight_bit else torch.float32)
    m.decode_step(ids[:, :6], cache)
    wrong = torch.randint(0, 100263, (3, 5))
    wrong[0, :2] = ids[0, 6:8]                       # sequence 0 keeps two of these, sequence 2 all that are right
    wrong[2] = ids[2, 6:11]
    m.decode_step(wrong, cache)
    cache.rollback(torch.tensor([3, 5, 0]))
    assert cache.positions.tolist() == [8, 6, 11] and cache.length == 11
    at = cache.positions
    nxt = torch.stack([ids[b, int(at[b]) : int(at[b]) + 4] for b in range(3)])
    step = m.decode_step(nxt, cache)
    for b in range(3):
        assert torch.allclose(step[b], full[b, int(at[b]) : int(at[b]) + 4], atol=2e-4, rtol=1e-4)
    cache.rollback(torch.tensor([12, 1, 0]))         # more than one step back
    assert cache.positions.tolist() == [0, 9, 15]
    step = m.decode_step(torch.stack([ids[0, :1], ids[1, 9:10], ids[2, 15:16]]), cache)
    for b, t in enumerate((0, 9, 15)):
        assert torch.allclose(step[b], full[b, t], atol=2e-4, rtol=1e-4)
    for bad in ([2, 0, 0], [-1, 0, 0]):
        with pytest.raises(ValueError, match="taken back"):
            cache.rollback(torch.tensor(bad))
    with pytest.raises(ValueError, match="one entry per sequence"):
        cache.rollback(torch.tensor([0, 0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.int8])
def test_steps_of_one_token_and_of_none(dtype, tiny_scale):
    m = tiny(tiny_scale, "nestor", 1)
    ids = torch.randint(0, 100263, (2, 3))
    flat, column = (m.init_kv_cache(2, 8, dtype=dtype) for _ in range(2))
    flat.rollback(torch.tensor([0, 0]))              # nothing was fed yet
    with pytest.raises(ValueError, match="taken back"):
        flat.rollback(torch.tensor([1, 0]))
    for t in range(3):
        a, b = m.decode_step(ids[:, t], flat), m.decode_step(ids[:, t : t + 1], column, torch.full((2, 1), t))
        assert a.shape == (2, 100263) and torch.equal(a, b)
    assert m.decode_step(ids[:, :0], flat).shape == (2, 0, 100263) and flat.length == 3


def test_logits_without_a_number_end_the_drafted_decoding(tiny_scale):
    m, draft = tiny(tiny_scale, "moe", 5), tiny(tiny_scale, "dense", 6)
    prompt = torch.randint(0, 100263, (2, 4))
    with torch.no_grad():
        m.head.weight.fill_(float("nan"))
    with pytest.raises(RuntimeError, match="no token to draw"):
        m.generate(prompt, 4, 0.8, torch.Generator().manual_seed(0), torch.int8, draft, 3)


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
def test_what_was_taken_back_leaves_no_trace_in_8_bits(code, tiny_scale):
    """The ops themselves: blocks are functions of their contents, so two decode states that hold the same tokens agree to
    the last bits of the surrounding arithmetic, whatever was tried in between."""

    m = tiny(tiny_scale, "nestor", 2)
    ids = torch.randint(0, 100263, (2, 90))
    straight, tried = (m.init_kv_cache(2, 120, dtype=code) for _ in range(2))
    for t in range(0, 80, 5):
        a = m.decode_step(ids[:, t : t + 5], straight)
        b = m.decode_step(ids[:, t : t + 5], tried)
        assert torch.isfinite(a).all() and torch.equal(a, b)
        m.decode_step(torch.randint(0, 100263, (2, 7)), tried)
        tried.rollback(torch.tensor([7, 7]))
    for x, y in zip(straight.blocks, tried.blocks):
        for u, v in zip(x, y):
            assert torch.equal(u.count, v.count)
            for l, n in enumerate(u.count.tolist()):
                b = -(-n // 64)
                assert torch.equal(u.kv.k_scale[l, :, :b], v.kv.k_scale[l, :, :b])
                assert torch.equal(u.kv.v_codes[l, :, :b].view(torch.uint8), v.kv.v_codes[l, :, :b].view(torch.uint8))


@pytest.mark.parametrize("cache_dtype", [torch.float32, torch.int8])
def test_greedy_decoding_with_drafts_is_the_models_own(cache_dtype, tiny_scale, monkeypatch):
    ExactCache(monkeypatch)
    m = tiny(tiny_scale, "nestor", 3)
    prompt = torch.randint(0, 100263, (3, 5))
    want = m.generate(prompt, 12)
    assert torch.equal(want, m.generate(prompt, 12, cache_dtype=cache_dtype))
    other = tiny(tiny_scale, "dense", 4)
    near = tiny(tiny_scale, "nestor", 3)             # the same weights, slightly off: some drafts are refused
    with torch.no_grad():
        for p in near.parameters():
            p.add_(torch.randn_like(p) * p.abs().mean() * 0.02)
    m.train()
    for draft, n in ((m, 4), (other, 1), (near, 3), (near, 6)):
        got = m.generate(prompt, 12, cache_dtype=cache_dtype, draft=draft, draft_tokens=n)
        assert torch.equal(want, got)
    assert m.training
    assert torch.equal(m.generate(prompt, 0, draft=other), prompt)
    for n in (0, 64):
        with pytest.raises(ValueError, match="draft_tokens"):
            m.generate(prompt, 2, draft=other, draft_tokens=n)
    with pytest.raises(ValueError, match="at least one token"):
        m.generate(prompt[:, :0], 2, draft=other)


def test_sampling_with_drafts_repeats_with_its_generator(tiny_scale):
    m, draft = tiny(tiny_scale, "moe", 5), tiny(tiny_scale, "dense", 6)
    prompt = torch.randint(0, 100263, (2, 4))
    runs = [m.generate(prompt, 7, 0.8, torch.Generator().manual_seed(s), torch.float8_e4m3fn, draft, 3) for s in (0, 0, 1)]
    assert runs[0].shape == (2, 11) and torch.equal(runs[0][:, :4], prompt)
    assert torch.equal(runs[0], runs[1]) and not torch.equal(runs[0], runs[2])


@pytest.mark.gpu
@pytest.mark.parametrize("compute", [None, torch.bfloat16])
def test_8_bit_decoding_runs_on_the_kernels(compute, tiny_scale):
    """The kernels against the statements of the same ops inside a model's steps, routing pinned. What may differ: in fp32
    a code where a key or value sits within 2^-20 of a rounding border (one step, 1/127 of a block's largest magnitude,
    in a rare entry), in bf16 the roundings of each layer's output (2^-8) as well."""

    m = tiny(tiny_scale, "nestor", 7).cuda()
    m.compute_dtype = compute
    ids = torch.randint(0, 100263, (4, 70), device="cuda")
    logits, tape = [], ops.RoutingTape()
    for kernels in (False, True):
        if kernels:
            cache = m.init_kv_cache(4, 80, dtype=torch.int8)
        else:
            with ops.oracle_ops():
                cache = m.init_kv_cache(4, 80, dtype=torch.int8)
        assert cache.blocks[0][0].kernels == kernels
        before = ops.launch_count()
        ops.set_routing_tape(tape, "replay" if kernels else "record")
        try:
            a = m.decode_step(ids[:, :64], cache)
            b = m.decode_step(ids[:, 64], cache)
            c = m.decode_step(ids[:, 65:70], cache)
        finally:
            ops.set_routing_tape(None)
        cache.rollback(torch.tensor([5, 0, 2, 1]))
        assert cache.positions.tolist() == [65, 70, 68, 69]
        assert (ops.launch_count() > before) == kernels
        logits.append(torch.cat((a, b.unsqueeze(1), c), dim=1))
    off = (logits[0] - logits[1]).abs().max() / logits[0].abs().max()
    assert off < (0.01 if compute is None else 0.05), off
    from nestor_b200.ops import _lib
    _lib.check_status(torch.device("cuda", 0))


@pytest.mark.gpu
def test_decoding_with_drafts_on_the_gpu(tiny_scale):
    m, draft = tiny(tiny_scale, "nestor", 8).cuda(), tiny(tiny_scale, "dense", 9).cuda()
    prompt = torch.randint(0, 100263, (3, 9), device="cuda")
    g = torch.Generator("cuda")
    runs = [m.generate(prompt, 10, 0.7, g.manual_seed(1), torch.int8, draft, 4) for _ in range(2)]
    assert runs[0].shape == (3, 19) and torch.equal(runs[0], runs[1]) and torch.equal(runs[0][:, :9], prompt)
    assert torch.equal(m.generate(prompt, 10, cache_dtype=torch.int8, draft=m, draft_tokens=3)[:, :9], prompt)
