"""The decoding operators on their own: the 8-bit key/value cache, attention over it, and the verification of drafts.

Each case is one call (or the few calls of one decode step that change the cache together) on inputs that a decode
loop has in hand. ``run`` computes it in plain torch operations, or, where ``own`` is set, through
``nestor_b200.ops``. A *list* is what one attention column has seen of one sequence (``list = column * B + sequence``);
a step's rows are packed by list and ``seg_start`` holds the bounds.

The cache of a list and head is cut into blocks of 64 entries with one fp32 scale each. A block's codes are stored in
units of 8 head dims x 64 entries, 32 lanes x 16 bytes, in the order the matrix instruction takes them:
``k``: lane ``(g, t)``, bytes ``(m, h, i)`` hold entry ``16m + 8h + g`` and dim ``8u + 2t + i``;
``v``: lane ``(g, t)``, bytes ``(m, h, i)`` hold entry ``16m + 8h + 2t + i`` and dim ``8u + g``.
"""

import math

import torch

own = False

BLOCK = 64
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------ cases
def listed():
    def append(name, **kw):
        return {"name": name, "op": "append", "columns": 8, "drop": 0, **kw}

    def attend(name, **kw):
        return {"name": name, "op": "attend", "columns": 8, "group": 1, "rows": 1, **kw}

    def verify(name, **kw):
        return {"name": name, "op": "verify", "vocab": 100263, **kw}

    return [
        # one new token of 64 sequences enters 3 of 8 columns: the cache update of every layer of every decode step
        append("append step", batch=64, chosen=3, heads=5, dim=40, rows=1, start=2048, type="bf16", code="int8"),
        # a 4096-token prompt of 8 sequences enters an empty cache at once
        append("append prompt", batch=8, chosen=6, heads=3, dim=40, rows=4096, start=0, type="bf16", code="e4m3"),
        # a drafted round of a dense model: four refused entries are taken back, five new ones follow
        append("append draft", batch=32, columns=1, chosen=1, heads=16, dim=60, rows=5, drop=4, start=1500, type="fp32", code="int8"),
        # the same in a wide column block with many short lists
        append("append take back", batch=64, chosen=8, heads=2, dim=80, rows=2, drop=1, start=300, type="fp16", code="e4m3"),
        # a single sequence at the beginning of its answer: latency counts
        attend("attend one", batch=1, chosen=8, heads=2, dim=40, length=512, type="bf16", code="int8"),
        # an ordinary evaluation batch at the pretraining length
        attend("attend batch", batch=16, chosen=5, heads=3, dim=40, length=2560, type="bf16", code="e4m3"),
        # many long sequences, the first block's three of eight columns: the largest read
        attend("attend long", batch=64, chosen=3, heads=5, dim=40, length=12288, type="bf16", code="int8"),
        # five drafted tokens a sequence against a dense model's cache
        attend("attend draft", batch=32, columns=1, chosen=1, rows=5, heads=16, dim=60, length=8192, type="fp16", code="int8"),
        # shared key heads of the widest head, full-precision queries
        attend("attend shared", batch=8, columns=1, chosen=1, heads=4, group=8, dim=128, length=20001, type="fp32", code="e4m3"),
        # greedy drafts (the draft model's own best tokens) of one sequence
        verify("verify one", batch=1, drafted=4, type="fp32", greedy=True),
        # sampled drafts of a batch, probabilities in 16 bits
        verify("verify batch", batch=64, drafted=8, type="bf16", greedy=False),
        # the largest batch
        verify("verify many", batch=256, drafted=4, type="fp32", greedy=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "verify"])
    kind, code = rng.choice(sorted(TYPES)), rng.choice(sorted(CODES))
    if op == "verify":
        vocab = rng.choice([100263, 50257, _log(rng, 300, 128001)])
        batch, drafted = _log(rng, 1, 256), rng.randint(0, 9)
        batch = max(1, min(batch, int(256 * 5 * 100263 / (vocab * (drafted + 1)))))
        return {"op": op, "vocab": vocab, "batch": batch, "drafted": drafted, "type": kind, "greedy": rng.random() < 0.3}
    columns = rng.choice([1, 1, 8, 8, 4])
    case = {"op": op, "batch": _log(rng, 1, 64), "columns": columns, "chosen": rng.randint(1, columns),
            "heads": rng.choice([1, 2, 3, 4, 5, 8, 16]), "dim": rng.choice([8, 24, 30, 40, 60, 64, 72, 80, 100, 128]),
            "type": kind, "code": code}
    if op == "append":
        # several blocks at once start at a block's first entry, as chunks of a prompt do
        long = rng.random() < 0.4
        case |= {"rows": _log(rng, 65, 4096) if long else _log(rng, 1, 64), "drop": 0 if long else rng.choice([0, 0, 1, 4, 16])}
        case["start"] = 64 * rng.randint(0, 16) if long else _log(rng, 17, 3000)
        most = 8 * 6 * 4096 * 3 * 40
        while case["batch"] > 1 and case["batch"] * case["chosen"] * case["rows"] * case["heads"] * case["dim"] > most:
            case["batch"] //= 2
        case["rows"] = max(1, min(case["rows"], most // (case["chosen"] * case["heads"] * case["dim"])))
        return case
    case |= {"rows": rng.choice([1, 1, 1, 2, 4, 5, 9]), "group": rng.choice([1, 1, 1, 2, 4, 8]), "length": _log(rng, 1, 30000)}
    most = 64 * 3 * 12288 * 5 * 40
    while case["batch"] > 1 and case["batch"] * columns * case["rows"] * case["length"] * case["heads"] * case["dim"] * case["group"] ** 0.5 > most:
        case["batch"] //= 2
    case["length"] = max(1, min(case["length"], int(most / (case["batch"] * columns * case["rows"] * case["heads"] * case["dim"]))))
    return case


# ----------------------------------------------------------------------------- inputs
def _rows_of_lists(case, g):
    """New rows of every list: each of a sequence's ``rows`` tokens enters ``chosen`` of its columns."""

    B, G, k, n = case["batch"], case["columns"], case["chosen"], case["rows"]
    order = torch.rand(B, n, G, generator=g, device="cuda").argsort(dim=-1)[..., :k]
    member = torch.zeros(B, n, G, device="cuda", dtype=torch.int32).scatter_(2, order, 1)
    return member.sum(1).t().reshape(-1).to(torch.int32)           # [G * B]


def _bounds(count):
    seg = torch.zeros(count.numel() + 1, dtype=torch.int32, device="cuda")
    seg[1:] = count.cumsum(0)
    return seg


def _read_rows(case):
    """Rows of the buffer that is read into: room for the older entries of every touched list's first block."""

    rows, old = case["batch"] * case["rows"] * case["chosen"], 0 if case["rows"] > BLOCK else BLOCK - 1
    return rows + old * min(rows, case["batch"] * case["columns"])


def _cache(case, lists, blocks, g, open_type):
    H, D = case["heads"], case["dim"]
    U = -(-D // 8)
    dtype, top = CODES[case["code"]]
    state = {}
    for x in ("k", "v"):
        codes = torch.randn(lists, H, blocks, U, 512, generator=g, device="cuda", dtype=torch.float16).mul_(0.3 * top)
        codes = codes.clamp_(-top, top)
        codes = codes.round_().to(torch.int8) if dtype == torch.int8 else codes.to(dtype)
        if D % 8:          # dims past the head's width hold zeros
            raw = codes.view(torch.int8).view(lists, H, blocks, U, 8, 4, 4, 2, 2)
            if x == "k":
                past = (8 * (U - 1) + 2 * torch.arange(4, device="cuda")[:, None] + torch.arange(2, device="cuda")) >= D
                raw[..., U - 1, :, :, :, :, :].masked_fill_(past[None, :, None, None, :], 0)
            else:
                past = (8 * (U - 1) + torch.arange(8, device="cuda")) >= D
                raw[..., U - 1, :, :, :, :, :].masked_fill_(past[:, None, None, None, None], 0)
        state[x + "_codes"] = codes
        state[x + "_scale"] = torch.rand(lists, H, blocks, generator=g, device="cuda").mul_(0.6).add_(0.7).mul_(3.0 / top)
        state[x + "_open"] = torch.randn(lists, H, 2, BLOCK, D, generator=g, device="cuda").to(open_type)
    return state


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, g)
    kind = TYPES[case["type"]]
    count = _rows_of_lists(case, g)
    L, H, D = count.numel(), case["heads"], case["dim"]
    seg = _bounds(count)
    rows = case["batch"] * case["rows"] * case["chosen"]
    s = {"case": case, "seg_start": seg, "rows": rows, "max_rows": case["rows"]}
    if case["op"] == "append":
        if case["rows"] > BLOCK:
            start = torch.full((L,), case["start"], dtype=torch.int32, device="cuda")
        else:
            start = torch.randint(case["start"] // 2, case["start"] + 1, (L,), generator=g, device="cuda", dtype=torch.int32)
        blocks = (case["start"] + case["rows"]) // BLOCK + 2
        s |= _cache(case, L, blocks, g, kind)
        s["k"] = torch.randn(rows, H, D, generator=g, device="cuda").to(kind)
        s["v"] = (torch.randn(rows, H, D, generator=g, device="cuda") * 0.5).to(kind)
        kept = (start - case["drop"]).clamp_min(0)
        s["start"] = kept
        # what is read back: the new entries with the older ones of the block that they fall into
        back = torch.where(count > 0, count + kept % BLOCK, 0).to(torch.int32)
        s["read_seg"], s["read_start"] = _bounds(back), (kept // BLOCK * BLOCK).to(torch.int32)
        s["read_rows"], s["read_used"] = _read_rows(case), int(back.sum())        # (rows behind the last list are zeros)
        return s
    base = torch.randint((case["length"] + 1) // 2, case["length"] + 1, (L,), generator=g, device="cuda", dtype=torch.int32)
    s["lengths"] = base + count
    s |= _cache(case, L, (case["length"] + case["rows"]) // BLOCK + 1, g, kind)
    spread = torch.randn(rows, H * case["group"], 1, generator=g, device="cuda").mul_(0.7).exp_()
    s["q"] = (torch.randn(rows, H * case["group"], D, generator=g, device="cuda") * 2.0 * spread).to(kind)
    s["scale"] = 1.0 / D
    return s


def _prepare_verify(case, g):
    B, n, V, kind = case["batch"], case["drafted"], case["vocab"], TYPES[case["type"]]
    logits = torch.randn(B, n + 1, V, generator=g, device="cuda").mul_(2.5)
    p = torch.softmax(logits, dim=-1).to(kind)
    s = {"case": case, "target_probs": p, "draft_probs": None}
    if case["greedy"]:
        near = logits[:, :n].add_(torch.randn(B, n, V, generator=g, device="cuda").mul_(0.1))
        s["draft_tokens"] = near.argmax(-1)
    else:
        near = logits[:, :n].add_(torch.randn(B, n, V, generator=g, device="cuda").mul_(0.5))
        s["draft_probs"] = q = torch.softmax(near, dim=-1).to(kind)
        s["draft_tokens"] = torch.multinomial(q.float().view(B * n, V), 1, generator=g).view(B, n) if n else torch.zeros(B, 0, dtype=torch.long, device="cuda")
    s["accept_u"] = torch.rand(B, n, generator=g, device="cuda")
    if case["greedy"]:
        s["accept_u"] *= 0.02          # (a target that nearly always agrees with the draft's best token)
    s["sample_u"] = torch.rand(B, generator=g, device="cuda")
    s["draft_len"] = torch.randint((n + 1) // 2, n + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    return s


# ------------------------------------------------------------------------ plain forms
def _natural(codes, which):
    """``[n, H, U, 512]`` codes of whole blocks as fp32 ``[n, H, 64, 8U]``."""

    n, H, U = codes.shape[:3]
    x = codes.reshape(n, H, U, 8, 4, 4, 2, 2)                                # u, g, t, m, h, i
    x = x.permute(0, 1, 5, 6, 3, 2, 4, 7) if which == "k" else x.permute(0, 1, 5, 6, 4, 7, 2, 3)
    return x.to(torch.float32).reshape(n, H, BLOCK, 8 * U)


def _stored(x, which):
    """The inverse of ``_natural`` on codes ``[n, H, 64, 8U]``."""

    n, H, _, W = x.shape
    U = W // 8
    if which == "k":
        return x.reshape(n, H, 4, 2, 8, U, 4, 2).permute(0, 1, 5, 4, 6, 2, 3, 7).reshape(n, H, U, 512)
    return x.reshape(n, H, 4, 2, 4, 2, U, 8).permute(0, 1, 6, 7, 4, 2, 3, 5).reshape(n, H, U, 512)


def _take(codes, *at):
    return codes.view(torch.uint8)[at].view(codes.dtype)


def _quantise(x, there, code):
    """``x [n, H, 64, D]`` fp32 with ``there [n, 64]`` the entries that are held -> codes and scales ``[n, H]``."""

    dtype, top = CODES[code]
    x = torch.where(there[:, None, :, None], x, 0.0)
    most = x.abs().amax(dim=(2, 3))
    most = torch.where(most < 2.0 ** -100, 0.0, most)          # (a block of such values holds zeros)
    fit = torch.where(most == 0, 0.0, torch.full_like(most, top) / most)
    y = (x * fit[:, :, None, None]).clamp(-top, top)
    return (y.round().to(torch.int8) if dtype == torch.int8 else y.to(dtype)), most / top


def _write_blocks(s, which, lists, block, x, there):
    D = x.shape[-1]
    codes, scale = _quantise(x, there, s["case"]["code"])
    full = torch.zeros(*codes.shape[:3], -(-D // 8) * 8, dtype=torch.uint8, device="cuda")
    full[..., :D] = codes.view(torch.uint8)
    s[which + "_codes"].view(torch.uint8)[lists, :, block] = _stored(full, which)
    s[which + "_scale"][lists, :, block] = scale


def _plain_truncate(s, lengths):
    lists = torch.nonzero(lengths % BLOCK > 0).flatten()
    block = (lengths[lists] // BLOCK).long()
    there = torch.arange(BLOCK, device="cuda") < (lengths[lists] % BLOCK)[:, None]
    for which in ("k", "v"):
        _write_blocks(s, which, lists, block, s[which + "_open"][lists, :, block % 2].float(), there)


def _plain_append(s):
    seg, start = s["seg_start"].long(), s["start"].long()
    count = seg[1:] - seg[:-1]
    lists = torch.nonzero(count > 0).flatten()
    first = start[lists] // BLOCK
    per = (s["max_rows"] + BLOCK - 1) // BLOCK + 1                                   # blocks that one list can touch
    entry = first[:, None, None] * BLOCK + torch.arange(per * BLOCK, device="cuda").view(1, per, BLOCK)
    begin, end = start[lists][:, None, None], (start + count)[lists][:, None, None]
    new = (entry >= begin) & (entry < end)
    row = torch.where(new, seg[:-1][lists][:, None, None] + entry - begin, 0)
    touched = (entry[:, :, 0] < end[:, :, 0]).flatten()
    at = lists[:, None].expand(-1, per).flatten()[touched]
    block = (first[:, None] + torch.arange(per, device="cuda")).flatten()[touched]
    new, row, entry = (t.flatten(0, 1)[touched] for t in (new, row, entry))
    last = (end[:, 0, 0] - 1)[:, None].expand(-1, per).flatten()[touched] // BLOCK
    there = entry < (last * 0 + end[:, 0, 0][:, None].expand(-1, per).flatten()[touched])[:, None]
    keep = new & (block >= last - 1)[:, None]
    kb, ke = torch.nonzero(keep, as_tuple=True)
    for which in ("k", "v"):
        rows, held = s[which], s[which + "_open"]
        x = torch.where(new[..., None, None], rows[row].float(), held[at, :, block % 2].transpose(1, 2).float())
        _write_blocks(s, which, at, block, x.transpose(1, 2), there)
        held[at[kb], :, (block % 2)[kb], ke] = rows[row[kb, ke]]


def _plain_read(s):
    seg, start = s["read_seg"].long(), s["read_start"].long()
    D, kind = s["case"]["dim"], TYPES[s["case"]["type"]]
    count = seg[1:] - seg[:-1]
    used = s["read_used"]
    lists = torch.repeat_interleave(torch.arange(count.numel(), device="cuda"), count, output_size=used)
    entry = start[lists] + torch.arange(used, device="cuda") - seg[:-1][lists]
    lead = entry % BLOCK == 0                                                      # one gather for each block
    which_block = lead.cumsum(0) - 1
    at, block = lists[lead], (entry // BLOCK)[lead]
    out = []
    for which in ("k", "v"):
        x = _natural(_take(s[which + "_codes"], at, slice(None), block), which)[..., :D]
        x = x * s[which + "_scale"][at, :, block][:, :, None, None]
        out.append(torch.zeros(s["read_rows"], x.shape[1], D, dtype=kind, device="cuda"))
        out[-1][:used] = x.transpose(1, 2)[which_block, entry % BLOCK].to(kind)
    return out


def _plain_attend(s):
    case, q = s["case"], s["q"]
    seg, lengths = s["seg_start"].long(), s["lengths"].long()
    count = seg[1:] - seg[:-1]
    R, H, gq, D = s["rows"], case["heads"], case["group"], case["dim"]
    lists = torch.repeat_interleave(torch.arange(count.numel(), device="cuda"), count, output_size=R)
    visible = lengths[lists] - (seg[1:][lists] - 1 - torch.arange(R, device="cuda"))
    nb = s["k_codes"].shape[2]
    # every list once, in fp32, then its (few) rows against it
    used = torch.unique(lists)
    slot = torch.searchsorted(used, lists)
    held = []
    for which in ("k", "v"):
        codes = _take(s[which + "_codes"], used)
        x = _natural(codes.transpose(1, 2).reshape(-1, H, *codes.shape[3:]), which)[..., :D]
        x = x.view(used.numel(), nb, H, BLOCK, D) * s[which + "_scale"][used].transpose(1, 2)[..., None, None]
        held.append(x.transpose(1, 2).reshape(used.numel(), H, nb * BLOCK, D))
    most = max(1, case["rows"])
    within = torch.arange(R, device="cuda") - seg[:-1][lists]
    qs = torch.zeros(used.numel(), H, most * gq, D, device="cuda")
    qs.view(used.numel(), H, most, gq, D)[slot, :, within] = q.float().view(R, H, gq, D)
    see = torch.zeros(used.numel(), most, dtype=torch.long, device="cuda")
    see[slot, within] = visible
    z = qs @ held[0].transpose(2, 3) * s["scale"]
    hidden = torch.arange(nb * BLOCK, device="cuda") >= see.repeat_interleave(gq, 1)[:, None, :, None]
    z = z.masked_fill(hidden, -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = (e @ held[1]) / torch.where(total == 0, 1.0, total)
    return o.view(used.numel(), H, most, gq, D)[slot, :, within].reshape(R, H * gq, D).to(q.dtype)


def _plain_verify(s):
    p, x, q, u = s["target_probs"], s["draft_tokens"].long(), s["draft_probs"], s["accept_u"]
    B, n, V = x.shape[0], x.shape[1], p.shape[-1]
    length = s["draft_len"].long()
    px = p[:, :n].gather(2, x.unsqueeze(-1)).squeeze(-1).float()
    qx = q.gather(2, x.unsqueeze(-1)).squeeze(-1).float() if q is not None else torch.ones_like(px)
    ok = (u * qx < px) & (torch.arange(n, device="cuda") < length[:, None])
    a = ok.long().cumprod(1).sum(1)
    b = torch.arange(B, device="cuda")
    row = p[b, a].float()
    if n:
        at = a.clamp_max(n - 1)
        if q is not None:
            less = q[b, at].float()
        else:
            less = torch.zeros_like(row).scatter_(1, x[b, at][:, None], math.inf)
        rest = torch.where(row > less, row - less, 0.0)
        rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, row)
        row = torch.where((a < length)[:, None], rest, row)
    total = row.double().cumsum(1)
    hit = total > s["sample_u"].double()[:, None] * total[:, -1:]
    token = torch.where(hit.any(1), hit.int().argmax(1), -1)
    return a.int(), token.int()


# --------------------------------------------------------------------------------- run
def _framework_cache(s):
    from nestor_b200 import ops
    return ops.KV8Cache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], s["k_open"], s["v_open"])


def run(s):
    op = s["case"]["op"]
    if own:
        from nestor_b200 import ops
        if op == "verify":
            return ops.verify_draft(s["target_probs"], s["draft_tokens"], s["draft_probs"], s["accept_u"], s["sample_u"], s["draft_len"])
        cache = _framework_cache(s)
        if op == "attend":
            return ops.kv8_attention(s["q"], cache, s["seg_start"], s["lengths"], s["scale"], max_rows=s["max_rows"])
        if s["case"]["drop"]:
            ops.kv8_truncate(cache, s["start"])
        ops.kv8_append(cache, s["k"], s["v"], s["seg_start"], s["start"], max_rows=s["max_rows"])
        k, v = ops.kv8_read(cache, s["read_seg"], s["read_start"], s["read_rows"], dtype=s["k"].dtype)
    else:
        if op == "verify":
            return _plain_verify(s)
        if op == "attend":
            return _plain_attend(s)
        if s["case"]["drop"]:
            _plain_truncate(s, s["start"])
        _plain_append(s)
        k, v = _plain_read(s)
    return {"k": k, "v": v, **{x + y: s[x + y] for x in ("k", "v") for y in ("_scale", "_open")}}


# -------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "verify":
        # the accepted prefix ends in a row of the target's; a refusal needs the draft's row beside it (about one
        # sequence in four has none); the sums take an addition for each value
        rows = 1 if case["greedy"] or not case["drafted"] else 1.75
        n = case["batch"] * case["vocab"]
        return {"bytes": n * rows * SIZE[case["type"]], "flops": n * (rows + 1)}
    H, D, rows = case["heads"], case["dim"], case["batch"] * case["rows"] * case["chosen"]
    if case["op"] == "append":
        old = 0 if case["rows"] > BLOCK else min(rows, case["batch"] * case["columns"]) * min(BLOCK // 2, case["start"])
        size = SIZE[case["type"]]
        # new rows in, the open block's older originals in, codes out; codes back in and values out
        return {"bytes": 2 * H * D * ((rows + old) * (size + 2) + _read_rows(case) * size), "flops": 4 * H * D * (rows + old)}
    lists = min(rows, case["batch"] * case["columns"])
    length = case["length"] * 0.75 + case["rows"] * case["chosen"] / case["columns"]
    cache = lists * length * H * (2 * D + 8 / BLOCK)
    return {"bytes": cache + 2 * rows * H * case["group"] * D * SIZE[case["type"]],
            "flops": 4 * rows * length * H * case["group"] * D}


# -------------------------------------------------------------------- 64-bit definition
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify":
        return None        # whole numbers: they have to be equal
    return _exact_attend(case, s) if case["op"] == "attend" else _exact_append(case, s)


def _positions(which, U):
    """Where entry ``e`` and dim ``d`` of a block stand among its bytes: ``[64, 8U]``."""

    e = torch.arange(BLOCK, device="cuda")[:, None]
    d = torch.arange(8 * U, device="cuda")[None, :]
    if which == "k":
        lane, byte = (e % 8) * 4 + (d % 8) // 2, (e // 16) * 4 + (e % 16 // 8) * 2 + d % 2
    else:
        lane, byte = (d % 8) * 4 + (e % 8) // 2, (e // 16) * 4 + (e % 16 // 8) * 2 + e % 2
    return (d // 8) * 512 + lane * 16 + byte


def _exact_list(s, which, l, length):
    """The first ``length`` entries of list ``l`` in 64 bits: ``[H, length, D]``."""

    D = s["case"]["dim"]
    codes = s[which + "_codes"]
    nb = -(-length // BLOCK)
    flat = codes[l, :, :nb].reshape(codes.shape[1], nb, -1)
    at = _positions(which, codes.shape[3])[:, :D]
    x = flat.view(torch.uint8)[:, :, at].view(codes.dtype).to(torch.float64)         # [H, nb, 64, D]
    x = x * s[which + "_scale"][l, :, :nb].double()[:, :, None, None]
    return x.reshape(codes.shape[1], nb * BLOCK, D)[:, :length]


def _exact_attend(case, s):
    if case["batch"] * case["columns"] > 2000:
        return None
    H, gq = case["heads"], case["group"]
    out = torch.zeros(s["rows"], H * gq, case["dim"], dtype=torch.float64, device="cuda")
    seg, lengths = s["seg_start"].tolist(), s["lengths"].tolist()
    for l, length in enumerate(lengths):
        n = seg[l + 1] - seg[l]
        if n == 0:
            continue
        k, v = (_exact_list(s, w, l, length).repeat_interleave(gq, 0) for w in ("k", "v"))
        for a in range(n):
            seen = length - (n - 1 - a)
            z = (k[:, :seen] * s["q"][seg[l] + a].double()[:, None]).sum(-1) * s["scale"]
            out[seg[l] + a] = (torch.softmax(z, -1)[..., None] * v[:, :seen]).sum(1)
    return out


def _exact_append(case, s):
    seg, start = s["seg_start"].tolist(), s["start"].tolist()
    rs = s["read_seg"].tolist()
    D, H = case["dim"], case["heads"]
    dtype, top = CODES[case["code"]]
    out = {}
    for which in ("k", "v"):
        values = torch.zeros(s["read_rows"], H, D, dtype=torch.float64, device="cuda")
        scales, held = s[which + "_scale"].double(), s[which + "_open"].double()

        def block(x):
            # a code is defined by the fp32 factor and the fp32 product (ties are common among 16-bit values, so the
            # two roundings belong to the definition); the value that it stands for is not rounded here
            most = x.abs().amax(dim=(0, 2))                                          # [H]
            fit = (top / torch.where(most == 0, math.inf, most)).float().double()
            y = (x * fit[None, :, None]).float()
            y = y.round().double() if dtype == torch.int8 else y.to(dtype).double()
            return y * (most / top)[None, :, None], most / top

        for l in range(len(start)):
            n, begin = seg[l + 1] - seg[l], start[l]
            b, old = begin // BLOCK, begin % BLOCK
            if case["drop"] and old:
                scales[l, :, b] = block(held[l, :, b % 2, :old].transpose(0, 1))[1]
            if n == 0:
                continue
            rows = s[which][seg[l] : seg[l + 1]].double()
            x = torch.cat([held[l, :, b % 2, :old].transpose(0, 1), rows])
            last = (begin + n - 1) // BLOCK
            for i in range(b, last + 1):
                part = x[(i - b) * BLOCK : (i - b + 1) * BLOCK]
                y, scale = block(part)
                scales[l, :, i] = scale
                values[rs[l] + (i - b) * BLOCK : rs[l] + (i - b) * BLOCK + part.shape[0]] = y
                if i >= last - 1:
                    skip = max(0, begin - i * BLOCK)
                    held[l, :, i % 2, skip : part.shape[0]] = part[skip:].transpose(0, 1)
        out |= {which: values, which + "_scale": scales, which + "_open": held}
    return {"k": out["k"], "v": out["v"], **{x + y: out[x + y] for x in ("k", "v") for y in ("_scale", "_open")}}
