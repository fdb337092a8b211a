"""What is measured of the operators around a 4-bit key/value cache: rotary positions with several axes,
quantising keys and values as they are written to a paged cache, reading them back, and attention over the
cache.  `own` selects between the plain forms (elementary torch operations in 32 or 64 bits) and the calls a
user makes of `afa_flash_attention_kernels`.

The cache is one uint8 tensor [pages, kv_heads, 2, page_size, d / 2 + d / 16] (index 2: keys, values).  A row
holds one token's head: d / 2 bytes of codes (byte j: channel 2j in the low half, 2j + 1 in the high half),
then for each group of 64 channels its step s and its minimum m in the 16-bit type of the model.  A code c
stands for s * c + m;  m = min(x),  s = round16((max(x) - min(x)) / 15),  c = clamp(round((x - m) / s), 0, 15)
with halves to even, c = 0 where s = 0.
"""

import math

import torch

own = False

GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # One decode step of a batch of long conversations: text positions, the same on all three axes.
        dict(name="rotary_step", op="rotary", batch=64, n=1, heads=32, kv_heads=8, d=128, rot=128, axes=3,
             interleaved=False, far=1000000, grad=False, dtype="bf16"),
        # The patches of two video clips before attention, time x height x width, neighbouring channels paired.
        dict(name="rotary_video", op="rotary", batch=2, n=8190, heads=32, kv_heads=32, d=64, rot=64, axes=3,
             interleaved=True, far=128, grad=False, dtype="fp16"),
        # A training step on mixed text and images: forward, and gradients of the queries and shared keys.
        dict(name="rotary_train", op="rotary", batch=4, n=4099, heads=32, kv_heads=8, d=128, rot=128, axes=3,
             interleaved=False, far=8192, grad=True, dtype="bf16"),
        # One new token for each of 128 sequences: written, and read back.
        dict(name="write_step", op="write", batch=128, n=1, length=4000, kv_heads=8, d=128, page=64,
             ragged=False, dtype="bf16"),
        # Eight prompts of unequal length in one padded batch: written, and read back for the prompt's attention.
        dict(name="write_prompt", op="write", batch=8, n=4096, length=4096, kv_heads=8, d=128, page=64,
             ragged=True, dtype="fp16"),
        # A few hundred tokens of context in small pages, brought back to 16 bits before the next chunk.
        dict(name="read_chunk", op="read", batch=3, length=777, kv_heads=4, d=64, page=16, dtype="bf16"),
        # A long document's whole cache brought back to 16 bits.
        dict(name="read_context", op="read", batch=1, length=131072, kv_heads=8, d=128, page=64, dtype="bf16"),
        # One short conversation: the latency of a single call.
        dict(name="decode_small", op="attend", batch=1, n=1, length=500, even=True, heads=32, kv_heads=8, d=128,
             page=64, causal=False, ragged=False, dtype="bf16"),
        # An ordinary serving batch with lengths spread evenly up to 8192.
        dict(name="decode_batch", op="attend", batch=32, n=1, length=8192, even=False, heads=32, kv_heads=8,
             d=128, page=64, causal=False, ragged=False, dtype="bf16"),
        # A few very long contexts.
        dict(name="decode_long", op="attend", batch=8, n=1, length=131072, even=True, heads=32, kv_heads=8,
             d=128, page=128, causal=False, ragged=False, dtype="bf16"),
        # Every query head with its own keys and values, small pages.
        dict(name="decode_mha", op="attend", batch=16, n=1, length=4001, even=False, heads=32, kv_heads=32, d=64,
             page=16, causal=False, ragged=False, dtype="fp16"),
        # Checking up to five proposed tokens a sequence at once, each seeing those before it.
        dict(name="verify", op="attend", batch=16, n=5, length=16384, even=False, heads=64, kv_heads=8, d=128,
             page=32, causal=True, ragged=True, dtype="fp16"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "write", "read", "attend", "attend"])
    d = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "rotary":
        kv = rng.choice([1, 2, 3, 4, 8, 16, 32])
        heads = kv * rng.choice([1, 2, 4, 7]) if kv <= 8 else kv
        n = _spread(rng, 1, 16384)
        most = 4 * 4099 * 40 * 128 // (n * (heads + kv) * d)
        return dict(op=op, batch=_spread(rng, 1, max(1, min(64, most))), n=n, heads=heads, kv_heads=kv, d=d,
                    rot=rng.choice([d // 2, d, d]), axes=rng.choice([1, 2, 3]), interleaved=rng.random() < 0.5,
                    far=_spread(rng, 16, 1000000), grad=rng.random() < 0.5, dtype=dtype)
    kv = rng.choice([1, 2, 4, 5, 8, 16, 32])
    page = rng.choice([16, 32, 64, 128])
    if op == "write":
        n = _spread(rng, 1, 16384)
        most = 8 * 4096 * 8 * 128 // (n * kv * d)
        return dict(op=op, batch=_spread(rng, 1, max(1, min(256, most))), n=n, length=n + rng.randrange(0, 500),
                    kv_heads=kv, d=d, page=page, ragged=rng.random() < 0.5, dtype=dtype)
    length = _spread(rng, 1, 131072)
    if op == "read":
        most = 131072 * 8 * 128 // (length * kv * d)
        return dict(op=op, batch=_spread(rng, 1, max(1, min(16, most))), length=length, kv_heads=kv, d=d,
                    page=page, dtype=dtype)
    n = rng.choice([1, 1, 2, 3, 5, 9])
    most = 8 * 131072 * 8 * 128 // (length * kv * d * (2 if n > 2 else 1))
    group = rng.choice([1, 2, 3, 4, 7, 8] if kv <= 8 else [1, 2])
    return dict(op=op, batch=_spread(rng, 1, max(1, min(96, most))), n=n, length=max(length, n),
                even=rng.random() < 0.3, heads=kv * group, kv_heads=kv, d=d, page=page, causal=rng.random() < 0.6,
                ragged=n > 1 and rng.random() < 0.5, dtype=dtype)


def _lengths(case):
    """Tokens in the cache for each sequence: all alike, or spread evenly from `length` downwards."""
    b, top = case["batch"], case["length"]
    if case["op"] != "attend" or case["even"]:
        return [top] * b
    return [max(case["n"], top - i * top // b) for i in range(b)]


def _new(case):
    """New tokens of each sequence: all `n`, or n, n - 1, ... spread down to about half (one at least)."""
    b, n = case["batch"], case["n"]
    if not case["ragged"]:
        return [n] * b
    return [max(1, n - i * n // (2 * b)) for i in range(b)]


def _row(d):
    return d // 2 + d // 16


def work(case):
    d = case["d"]
    if case["op"] == "rotary":
        rows = case["batch"] * case["n"] * (case["heads"] + case["kv_heads"])
        times = 2 if case["grad"] else 1
        table = case["batch"] * case["n"] * case["axes"] * 8 + case["rot"] * 2
        return {"bytes": times * (rows * d * 4 + table), "flops": times * rows * case["rot"] * 3}
    if case["op"] == "write":
        rows = sum(_new(case)) * case["kv_heads"] * 2
        padded = case["batch"] * case["n"] * case["kv_heads"] * 2
        return {"bytes": rows * (2 * d + 2 * _row(d)) + padded * 2 * d, "flops": rows * d * 8}
    if case["op"] == "read":
        rows = sum(_lengths(case)) * case["kv_heads"] * 2
        return {"bytes": rows * (2 * d + _row(d)), "flops": rows * d * 2}
    tokens = sum(_lengths(case))
    q = case["batch"] * case["n"] * case["heads"]
    pairs = sum(x * n for x, n in zip(_lengths(case), _new(case))) * case["heads"]
    return {"bytes": tokens * case["kv_heads"] * 2 * _row(d) + q * (4 * d + 4), "flops": 4 * pairs * d}


# ---------------------------------------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------------------------------------
def _rotary_inputs(case, gen):
    dt, b, n, d = DTYPES[case["dtype"]], case["batch"], case["n"], case["d"]
    pairs = case["rot"] // 2
    axes = case["axes"]
    sections = [pairs // axes] * axes
    sections[0] += pairs - sum(sections)
    # one ladder of frequencies for each axis
    inv = torch.cat([10000.0 ** (-torch.arange(s, dtype=torch.float64) / s) for s in sections]).float().cuda()
    if n == 1:
        # a text token far into the conversation: the same position on every axis
        pos = torch.randint(0, case["far"] + 1, (1, b, 1), generator=gen, device="cuda").expand(axes, b, 1).contiguous()
    elif axes == 1:
        start = torch.randint(0, max(1, case["far"] - n) + 1, (b, 1), generator=gen, device="cuda")
        pos = (start + torch.arange(n, device="cuda")).view(1, b, n)
    else:
        # a grid of patches: the last axis runs fastest, the first one slowest, from a start of its own
        side = max(1, int(round(n ** (1.0 / axes))))
        i = torch.arange(n, device="cuda")
        cols = []
        for a in range(axes):
            step = side ** (axes - 1 - a)
            cols.append(i // step if a == 0 else i // step % side)
        start = torch.randint(0, case["far"] + 1, (axes, b, 1), generator=gen, device="cuda")
        pos = torch.stack(cols)[:, None, :] + start
    make = lambda h: torch.randn(b, n, h, d, generator=gen, device="cuda").to(dt)
    state = dict(q=make(case["heads"]), k=make(case["kv_heads"]), positions=pos, inv_freq=inv, sections=sections)
    if case["grad"]:
        state.update(dq=make(case["heads"]), dk=make(case["kv_heads"]))
    return state


def _keys(shape, gen, dt):
    """Keys as models have them: channels with an offset of their own."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x += 1.5 * torch.randn(shape[-2:], generator=gen, device="cuda")
    return x.to(dt)


def _pages(case, lengths, gen):
    """Page table int32 [batch, most pages] (-1 behind a sequence's last page) and the number of pages."""
    page = case["page"]
    need = [-(-x // page) for x in lengths]
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    return table, total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "rotary":
        state = _rotary_inputs(case, gen)
        state["case"] = case
        return state
    dt, b, d, kv = DTYPES[case["dtype"]], case["batch"], case["d"], case["kv_heads"]
    lengths = _lengths(case)
    table, total = _pages(case, lengths, gen)
    # pages in use before hold anything
    cache = torch.randint(0, 256, (total, kv, 2, case["page"], _row(d)), generator=gen, device="cuda", dtype=torch.uint8)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    state = dict(case=case, cache=cache, page_table=table, kv_lens=lens)
    if case["op"] == "write":
        n = case["n"]
        state.update(k=_keys((b, n, kv, d), gen, dt), v=torch.randn(b, n, kv, d, generator=gen, device="cuda").to(dt))
        state["new_lens"] = torch.tensor(_new(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
        return state
    # a filled cache: sequence after sequence, 65536 tokens at a time
    page = case["page"]
    for i, length in enumerate(lengths):
        for t0 in range(0, length, 65536):
            t1 = min(length, t0 + 65536)
            pos = torch.arange(t0, t1, device="cuda")
            ids = table[i, pos // page].long()
            cache[ids, :, 0, pos % page] = _quantise(_keys((t1 - t0, kv, d), gen, dt), torch.float32)
            v = torch.randn(t1 - t0, kv, d, generator=gen, device="cuda").to(dt)
            cache[ids, :, 1, pos % page] = _quantise(v, torch.float32)
    if case["op"] == "attend":
        state["q"] = torch.randn(b, case["n"], case["heads"], d, generator=gen, device="cuda").to(dt)
        state["new_lens"] = torch.tensor(_new(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    return state


# ---------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    if case["op"] == "rotary":
        return _plain_rotary(case, state)
    if case["op"] == "write":
        _plain_write(case, state)
        return _plain_read(case, state, case["n"], state["new_lens"])
    if case["op"] == "read":
        return _plain_read(case, state, case["length"], None)
    return _plain_attend(case, state)


def _own(case, s):
    import afa_flash_attention_kernels as fa

    if case["op"] == "rotary":
        if not case["grad"]:
            q, k = fa.rotary(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"], case["interleaved"])
            return {"q": q, "k": k}
        x, y = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
        q, k = fa.rotary(x, y, s["positions"], s["inv_freq"], s["sections"], case["interleaved"])
        dq, dk = torch.autograd.grad((q, k), (x, y), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    dt = DTYPES[case["dtype"]]
    if case["op"] == "write":
        fa.cache4_write(s["k"], s["v"], s["cache"], s["page_table"], s["kv_lens"], new_lens=s["new_lens"])
        k, v = fa.cache4_read(s["cache"], s["page_table"], s["kv_lens"], case["n"], dt, new_lens=s["new_lens"])
        return {"k": k, "v": v}
    if case["op"] == "read":
        k, v = fa.cache4_read(s["cache"], s["page_table"], s["kv_lens"], case["length"], dt)
        return {"k": k, "v": v}
    o, lse = fa.forward_cache4(s["q"], s["cache"], s["page_table"], s["kv_lens"], causal=case["causal"],
                               return_lse=True, new_lens=s["new_lens"])
    return {"o": o, "lse": lse}


def _plain_rotary(case, s):
    axis = torch.cat([torch.full((m,), a, device="cuda") for a, m in enumerate(s["sections"])])
    # angles of far positions in 64 bits: [batch, n, pairs]
    angle = s["positions"].double()[axis].permute(1, 2, 0) * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, :, None, :], angle.sin().float()[:, :, None, :]
    out = {"q": _rotate(case, s["q"], cos, sin), "k": _rotate(case, s["k"], cos, sin)}
    if case["grad"]:  # the transpose of a rotation is the rotation back
        out["dq"] = _rotate(case, s["dq"], cos, -sin)
        out["dk"] = _rotate(case, s["dk"], cos, -sin)
    return out


def _rotate(case, x, cos, sin):
    rot = case["rot"]
    out = x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:rot:2].float(), x[..., 1:rot:2].float()
        out[..., 0:rot:2] = (a * cos - b * sin).to(x.dtype)
        out[..., 1:rot:2] = (b * cos + a * sin).to(x.dtype)
    else:
        a, b = x[..., :rot // 2].float(), x[..., rot // 2:rot].float()
        out[..., :rot // 2] = (a * cos - b * sin).to(x.dtype)
        out[..., rot // 2:rot] = (b * cos + a * sin).to(x.dtype)
    return out


def _quantise(x, wide):
    """Rows of the cache, uint8 [..., d / 2 + d / 16], for x [..., d]."""
    g = x.unflatten(-1, (-1, GROUP)).to(wide)
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = ((high - low) / 15).to(x.dtype)
    wide_step = step.to(wide)
    code = torch.where(wide_step > 0, (g - low) / wide_step, torch.zeros_like(g)).round_().clamp_(0, 15).to(torch.uint8)
    code = code.flatten(-2)
    packed = code[..., 0::2] | code[..., 1::2] << 4
    pairs = torch.cat([step, low.to(x.dtype)], -1).flatten(-2).contiguous()
    return torch.cat([packed, pairs.view(torch.uint8)], -1)


def _values(rows, dt, d):
    """What rows of the cache stand for, in 32 bits: [..., d]."""
    packed = rows[..., :d // 2]
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP)).float()
    pairs = rows[..., d // 2:].contiguous().view(dt).unflatten(-1, (-1, 2)).float()
    return (code * pairs[..., :1] + pairs[..., 1:]).flatten(-2)


def _rows_of(case, s, n, new):
    """For new row i of sequence b: whether it is one, its page and its place in the page, [batch, n] each."""
    i = torch.arange(n, device="cuda")
    fresh = torch.full_like(s["kv_lens"], n) if new is None else new
    pos = (s["kv_lens"] - fresh)[:, None] + i
    there = (i < fresh[:, None]) & (pos >= 0)
    pos = torch.where(there, pos, torch.zeros_like(pos)).long()
    ids = s["page_table"].long().gather(1, pos // case["page"])
    return there, torch.where(there, ids, torch.zeros_like(ids)), pos % case["page"]


def _plain_write(case, s):
    there, ids, place = _rows_of(case, s, case["n"], s["new_lens"])
    for which, x in ((0, s["k"]), (1, s["v"])):
        rows = _quantise(x, torch.float64)
        if s["new_lens"] is None:
            s["cache"][ids, :, which, place] = rows
        else:
            s["cache"][ids[there], :, which, place[there]] = rows[there]


def _plain_read(case, s, n, new):
    there, ids, place = _rows_of(case, s, n, new)
    out = {}
    for name, which in (("k", 0), ("v", 1)):
        x = _values(s["cache"][ids, :, which, place], DTYPES[case["dtype"]], case["d"])
        out[name] = torch.where(there[:, :, None, None], x, torch.zeros_like(x)).to(DTYPES[case["dtype"]])
    return out


def _plain_attend(case, s):
    q, lens = s["q"], s["kv_lens"]
    b, n, heads, d = q.shape
    kv, page = case["kv_heads"], case["page"]
    dt = DTYPES[case["dtype"]]
    ids = s["page_table"].long().clamp(min=0)
    length = ids.shape[1] * page
    j = torch.arange(length, device="cuda")
    there = (j < lens[:, None])[:, None, :, None]  # [batch, 1, tokens, 1]
    fresh = torch.full_like(lens, n) if s["new_lens"] is None else s["new_lens"]
    i = torch.arange(n, device="cuda")
    last = lens[:, None] - fresh[:, None] + i if case["causal"] else (lens - 1)[:, None].expand(b, n)
    sees = (j <= last[..., None]) & (j < lens[:, None, None]) & (i < fresh[:, None])[..., None]
    sees = sees[:, None, :, None, :]  # [batch, 1, n, 1, tokens]

    def side(which):
        rows = s["cache"][:, :, which][ids]  # [batch, pages, kv, page, row]
        x = _values(rows.transpose(1, 2).reshape(b, kv, length, -1), dt, d)
        return torch.where(there, x, torch.zeros_like(x))

    k = side(0)
    qs = q.float().view(b, n, kv, heads // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d)
    score = (qs @ k.transpose(2, 3)).view(b, kv, n, heads // kv, length) * (1 / math.sqrt(d))
    del k
    score = torch.where(sees, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = (score - top).exp()
    del score
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, kv, -1, length) @ side(1)).view(b, kv, n, heads // kv, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log()).squeeze(-1)  # -inf where nothing is seen
    o = o.permute(0, 2, 1, 3, 4).reshape(b, n, heads, d)
    return {"o": o.to(dt), "lse": lse.permute(0, 1, 3, 2).reshape(b, heads, n)}


# ---------------------------------------------------------------------------------------------------------
# The definitions in 64 bits, written apart from the forms above
# ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    if case["op"] == "write":
        return _exact_write(case, s)
    if case["op"] == "read":
        lens = [case["length"]] * case["batch"]
        got = [_exact_context(case, s, i, t, 0) + _exact_context(case, s, i, t, 1) for i, t in enumerate(lens)]
        return {"k": torch.stack([g[0] for g in got]), "v": torch.stack([g[1] for g in got])}
    return _exact_attend(case, s)


def _exact_rotary(case, s):
    rot = case["rot"]
    first, parts = 0, []
    for a, m in enumerate(s["sections"]):
        parts.append(s["positions"][a].double()[..., None] * s["inv_freq"][first:first + m].double())
        first += m
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.cat(parts, -1))[:, :, None, :]

    def rotated(x, turn):
        x = x.double()
        head, tail = x[..., :rot], x[..., rot:]
        if case["interleaved"]:
            z = torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * turn
            return torch.cat([torch.view_as_real(z).flatten(-2), tail], -1)
        z = torch.complex(*head.chunk(2, -1)) * turn
        return torch.cat([z.real, z.imag, tail], -1)

    out = {"q": rotated(s["q"], turn), "k": rotated(s["k"], turn)}
    if case["grad"]:
        out.update(dq=rotated(s["dq"], turn.conj()), dk=rotated(s["dk"], turn.conj()))
    return out


def _exact_write(case, s):
    dt = DTYPES[case["dtype"]]
    new = torch.tensor(_new(case), device="cuda")
    real = (torch.arange(case["n"], device="cuda") < new[:, None])[:, :, None, None]
    out = {}
    for name in ("k", "v"):
        x = s[name].double()
        parts = []
        for c in range(0, case["d"], GROUP):
            g = x[..., c:c + GROUP]
            low = g.min(-1, keepdim=True).values
            step = ((g.max(-1, keepdim=True).values - low) / 15).to(dt).double()
            code = torch.clamp(torch.round((g - low) / torch.where(step == 0, torch.ones_like(step), step)), 0, 15)
            parts.append(low + step * torch.where(step == 0, torch.zeros_like(code), code))
        out[name] = torch.where(real, torch.cat(parts, -1), torch.zeros_like(x))
    return out


def _exact_context(case, s, i, length, which):
    """One sequence's keys or values in 64 bits, as a tuple of one tensor [length, kv, d]."""
    d, page = case["d"], case["page"]
    pages = s["page_table"][i, :-(-length // page)].tolist()
    rows = torch.cat([s["cache"][p, :, which] for p in pages], 1)[:, :length]  # [kv, length, row]
    x = torch.empty(*rows.shape[:2], d, dtype=torch.float64, device="cuda")
    x[..., 0::2] = (rows[..., :d // 2] % 16).double()
    x[..., 1::2] = (rows[..., :d // 2] // 16).double()
    params = rows[..., d // 2:].contiguous().view(DTYPES[case["dtype"]]).double()
    for g in range(d // GROUP):
        x[..., g * GROUP:(g + 1) * GROUP].mul_(params[..., 2 * g, None]).add_(params[..., 2 * g + 1, None])
    return (x.transpose(0, 1),)


def _exact_attend(case, s):
    b, n, heads, d = s["q"].shape
    kv = case["kv_heads"]
    o = torch.zeros(b, n, heads, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, heads, n), -math.inf, dtype=torch.float64, device="cuda")
    for i, (length, fresh) in enumerate(zip(_lengths(case), _new(case))):
        k, v = (_exact_context(case, s, i, length, w)[0].transpose(0, 1) for w in (0, 1))
        for t in range(fresh):
            upto = length - fresh + t + 1 if case["causal"] else length
            if upto <= 0:
                continue
            x = s["q"][i, t].double().view(kv, heads // kv, d)
            score = torch.einsum("kgd,ktd->kgt", x, k[:, :upto]) / math.sqrt(d)
            lse[i, :, t] = torch.logsumexp(score, -1).flatten()
            o[i, t] = torch.einsum("kgt,ktd->kgd", torch.softmax(score, -1), v[:, :upto]).reshape(heads, d)
    return {"o": o, "lse": lse}
