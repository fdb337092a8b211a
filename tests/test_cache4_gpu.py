"""The paged 4-bit cache on the GPU: the writer's bytes against exact arithmetic,
the reader's values, and attention over the cache against a 64-bit oracle.

Tolerances.
* Writer: none; codes, steps and minima are equal.
* Reader: s c + m rounded once: half a step of the value's type.
* Attention: with p the weights of a row, the output is rounded once (eps / 2
  relative) from sum_t p_t (s' c' + m'), where p s' was rounded to fp16 (2^-11
  relative) and each p is off by twice its score's error and that of the base-2
  exponential (2^-21).  A score is a sum of at most 8 matrix instructions and 6
  fp32 steps over terms that add up to `reach` in magnitude; each is charged a
  whole unit of the 23rd bit: 14 * 2^-23 < 2^-19 reach.  l and the sums over the
  tokens add below 2^-16 (at most 2^12 fp32 additions a lane, each half a unit of the
  24th bit).  So
      |O - O64| <= eps / 2 |O64| + (2^-11 + 2^-18 reach + 2^-15) weight
  with weight = sum_t p_t (s' c' + |m'|), and
      |lse - lse64| <= 2^-19 reach + 2^-15 + 2^-22 |lse64|.
"""

import math

import pytest
import torch

import afa_flash_attention_kernels as fa
from oracle import cache4_oracle as oc

pytestmark = pytest.mark.gpu

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def pages(lens, page, seed=0, spare=2):
    """Page table (-1 behind a sequence's last page) over shuffled pages, on the CPU."""
    need = [max(1, -(-n // page)) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def noise_cache(n_pages, heads, page, d, seed=0):
    """Pages that hold anything, NaN and infinite steps among it."""
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, 256, (n_pages, heads, 2, page, d // 2 + d // 16), generator=g, dtype=torch.uint8)
    c[:, :, :, ::3, d // 2:] = 255
    return c


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


def filled(lens, heads, d, page, dtype, seed=0, k_scale=1.0, v_scale=1.0, offset=1.0):
    """(cache, table) on the CPU with every sequence's tokens quantised by the oracle; other rows are noise."""
    table, n_pages = pages(lens, page, seed)
    cache = noise_cache(n_pages, heads, page, d, seed)
    g = torch.Generator().manual_seed(seed + 1)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        t = torch.arange(n)
        for w, scale in ((0, k_scale), (1, v_scale)):
            x = torch.randn(n, heads, d, generator=g) * scale
            if w == 0:
                x += offset * torch.randn(heads, d, generator=g)
            rows = oc.pack_rows(*oc.quantise64(x.to(dtype), dtype), dtype)
            cache[table[b, t // page].long(), :, w, t % page] = rows
    return cache, table


# --- writer ----------------------------------------------------------------------------------------------
def hard_rows(dtype, d, seed):
    """Rows where rounding is decided close: halves, constants, far ranges, tiny and large values."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(96, d, generator=g)
    x[0] = 0
    x[1] = -3.5
    x[2] = torch.arange(d) % 31 / 2.0  # range 15: halves of a step
    x[3] = torch.arange(d) % 16 * 0.25 - 1
    x[4] = 1e-7 * x[4]
    x[5] = 1e4 * x[5]
    x[6, ::2] *= 1e-5
    x[7] = x[7] * 1e-3 + 100
    x[8] = (torch.arange(d) % 4) * 2.0 ** -24  # fp16: subnormal steps, a step of 0
    x[9] = (torch.arange(d) % 64) * 2.0 ** -24
    x[10, 1:] = 0
    x[11:40] = torch.randint(-8, 9, (29, d), generator=g) / 4.0  # few bits: many exact ties
    x[40:60] = torch.randint(0, 200, (20, d), generator=g).float()
    y = x.to(dtype)
    if dtype == torch.bfloat16:
        y[60] = y[60] * 1e37
        y[61] = (y[61].double() * 1e-39).to(dtype)
        y[62, 0], y[62, 1] = 3e38, -1e-30
        y[63, 0], y[63, 1] = -6.5, 1e-30  # next to a border of the step 1
        y[63, 2] = 8.5
    return y


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_written_bytes_are_exact(dtype, d):
    x = hard_rows(dtype, d, 1).view(1, 96, 1, d)
    table, n_pages = pages([96], 32)
    cache = noise_cache(n_pages, 1, 32, d).cuda()
    fa.cache4_write(x.cuda(), x.flip(1).cuda(), cache, table.cuda(), ints([96]).cuda())
    fa.check_status(0)
    rows = oc.sequence_rows(cache.cpu(), table, 0, 96)
    want = oc.quantise_exact(x[0, :, 0], dtype)
    for got, exp in ((rows[0, :, 0], want), (rows[1, :, 0], tuple(t.flip(0) for t in want))):
        for a, b, what in zip(oc.unpack_rows(got, dtype), exp, ("codes", "s", "m")):
            assert torch.equal(a, b), (what, (a != b).nonzero()[:5].tolist())


WRITES = [
    # lens after the write, n, new_lens, heads, d, page, dtype
    ([1], 1, None, 1, 64, 16, torch.float16),
    ([1, 500, 64, 65], 1, None, 8, 128, 64, torch.bfloat16),
    ([300, 257, 1000], 257, None, 3, 64, 128, torch.bfloat16),
    ([40, 7, 128, 129], 40, [40, 7, 0, 1], 2, 128, 16, torch.float16),
    ([1300], 1200, None, 5, 128, 256, torch.float16),
    ([0, 30], 9, [0, 5], 1, 64, 32, torch.bfloat16),
]


@pytest.mark.parametrize("case", WRITES, ids=lambda c: f"n{c[1]}-h{c[3]}-d{c[4]}-p{c[5]}")
def test_write_and_read_back(case):
    lens, n, new, heads, d, page, dtype = case
    B = len(lens)
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(B, n, heads, d, generator=g).to(dtype) for _ in range(2))
    table, n_pages = pages(lens, page, n)
    before = noise_cache(n_pages, heads, page, d)
    cache = before.cuda()
    dev = [t.cuda() if t is not None else None for t in (table, ints(lens), ints(new) if new else None)]
    for t in (k, v):  # padding rows may hold anything
        for b in range(B):
            t[b, (new[b] if new else n):] = math.nan
    fa.cache4_write(k.cuda(), v.cuda(), cache, dev[0], dev[1], dev[2])
    expect = before.clone()
    for b in range(B):
        m = new[b] if new else n
        for i in range(m):
            t = lens[b] - m + i
            for w, x in ((0, k), (1, v)):
                expect[table[b, t // page], :, w, t % page] = oc.pack_rows(*oc.quantise64(x[b, i], dtype), dtype)
    assert torch.equal(cache.cpu(), expect)  # the new rows, and nothing else
    kr, vr = fa.cache4_read(cache, dev[0], dev[1], n, dtype, dev[2])
    fa.check_status(0)
    for b in range(B):
        m = new[b] if new else n
        rows = oc.sequence_rows(expect, table, b, lens[b])[:, lens[b] - m:]
        for got, r in ((kr, rows[0]), (vr, rows[1])):
            c, s, mn = oc.unpack_rows(r, dtype)
            want = c * s.repeat_interleave(64, -1) + mn.repeat_interleave(64, -1)
            x = got[b, :m].cpu().double()
            # rounding once leaves half a step of the value's own binade; |x| covers a value rounded up to a power of two
            assert torch.all((x - want).abs() <= torch.finfo(dtype).eps / 2 * x.abs() + TINY[dtype])
            assert not got[b, m:].any()


def test_non_finite_groups_read_back_as_nan():
    x = torch.randn(1, 6, 1, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    x[0, 0, 0, 5] = math.nan
    x[0, 1, 0, 70] = math.inf
    x[0, 2, 0, 0] = -math.inf
    x[0, 3, 0, 64], x[0, 3, 0, 65] = 3e38, -3e38  # the range passes fp32
    table, lens = ints([[1]]).cuda(), ints([6]).cuda()
    cache = torch.zeros(2, 1, 2, 16, 72, dtype=torch.uint8, device="cuda")
    fa.cache4_write(x.cuda(), x.cuda(), cache, table, lens)
    k, v = fa.cache4_read(cache, table, lens, 6, torch.bfloat16)
    bad = torch.zeros(6, 2, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 0] = bad[3, 1] = True
    for t in (k, v):
        nan = torch.isnan(t[0, :, 0].cpu().view(6, 2, 64))
        assert torch.equal(nan.all(-1), bad) and torch.equal(nan.any(-1), bad)


def test_strided_inputs_outputs_and_pages():
    g = torch.Generator().manual_seed(3)
    kv = torch.randn(2, 50, 2, 3, 64, generator=g).half().cuda()  # packed keys and values
    layers = torch.zeros(12, 4, 3, 2, 16, 36, dtype=torch.uint8, device="cuda")  # pages of four layers side by side
    table = ints([[0, 3, 5, 7, -1], [11, 2, 1, 9, -1]]).cuda()[:, :4]
    lens = ints([50, 50]).cuda()
    dense = torch.zeros(12, 3, 2, 16, 36, dtype=torch.uint8, device="cuda")
    fa.cache4_write(kv[:, :, 0], kv[:, :, 1], layers[:, 2], table, lens)
    fa.cache4_write(kv[:, :, 0].contiguous(), kv[:, :, 1].contiguous(), dense, table, lens)
    assert torch.equal(layers[:, 2], dense) and not layers[:, [0, 1, 3]].any()
    out = torch.full((2, 50, 2, 3, 64), 7.0, dtype=torch.float16, device="cuda")
    k, v = fa.cache4_read(dense, table, lens, 50, torch.float16)
    a, b = fa.cache4_read(layers[:, 2], table, lens, 50, torch.float16, None, out[:, :, 0], out[:, :, 1])
    assert a.data_ptr() == out.data_ptr() and torch.equal(a, k) and torch.equal(b, v)
    # one row repeated over the batch
    rep = kv[:1, :, 0].expand(2, 50, 3, 64)
    fa.cache4_write(rep, rep, dense, table, lens)
    k, v = fa.cache4_read(dense, table, lens, 50, torch.float16)
    assert torch.equal(k[0], k[1]) and torch.equal(k, v)
    q = torch.randn(2, 2, 6, 64, generator=g).half().cuda()
    fa.cache4_write(kv[:, :, 0], kv[:, :, 1], dense, table, lens)
    o, lse = fa.forward_cache4(q, dense, table, lens, None, True, None, True)
    o2, lse2 = fa.forward_cache4(q, layers[:, 2], table, lens, None, True, None, True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    wide = torch.zeros(2, 6, 2, 2, 64, dtype=torch.float16, device="cuda")  # head-major q, strided o
    qh = q.transpose(1, 2).contiguous().transpose(1, 2)
    view = wide[:, :, :, 1].transpose(1, 2)
    o3, _ = fa.forward_cache4(qh, dense, table, lens, view, True)
    assert o3.data_ptr() == view.data_ptr() and torch.equal(o3, o) and not wide[:, :, :, 0].any()


# --- attention -------------------------------------------------------------------------------------------
def check_attention(q, cache, table, lens, causal, new=None, scale=None, got=None):
    B, N = q.shape[:2]
    if got is None:
        got = fa.forward_cache4(q.cuda(), cache.cuda(), table.cuda(), ints(lens).cuda(), None, causal, scale, True,
                                ints(new).cuda() if new else None)
        fa.check_status(0)
    o, lse = (t.cpu().double() for t in got)
    want, want_lse, weight, reach = oc.attention64(q, cache, table, lens, causal, scale, new)
    eps = torch.finfo(q.dtype).eps
    tol = want.abs() * eps / 2 + (2.0 ** -11 + 2.0 ** -18 * reach[..., None] + 2.0 ** -15) * weight + TINY[q.dtype]
    err = (o - want).abs()
    assert torch.all(err <= tol), f"largest error over tolerance {(err / tol).max().item():.3f}"
    fin = torch.isfinite(want_lse)
    assert torch.equal(torch.isfinite(lse), fin) and torch.all(lse[~fin] == -math.inf)
    tol = 2.0 ** -19 * reach.transpose(1, 2) + 2.0 ** -15 + 2.0 ** -22 * want_lse.abs()
    assert torch.all(((lse - want_lse).abs() <= tol)[fin])
    return o, lse


ATTEND = [
    # lens, n, new_lens, H, HK, d, page, causal, dtype
    ([1], 1, None, 1, 1, 64, 16, False, torch.float16),
    ([1], 1, None, 8, 1, 128, 64, True, torch.bfloat16),
    ([15, 16, 17, 31, 32, 33], 1, None, 4, 4, 64, 16, False, torch.bfloat16),
    ([127, 128, 129, 0, 500], 1, None, 8, 2, 128, 32, False, torch.float16),
    ([0, 0], 2, None, 2, 1, 64, 16, True, torch.float16),
    ([1000, 3, 257], 1, None, 32, 8, 128, 64, False, torch.bfloat16),
    ([700], 1, None, 7, 1, 128, 128, False, torch.float16),
    ([300, 40], 5, None, 8, 2, 128, 16, True, torch.bfloat16),
    ([300, 40], 5, None, 8, 2, 64, 256, False, torch.float16),
    ([64, 3, 90], 7, [7, 3, 1], 6, 3, 64, 32, True, torch.bfloat16),
    ([64, 0, 90], 7, [7, 0, 0], 6, 3, 128, 32, False, torch.float16),
    ([2, 1], 4, None, 2, 2, 64, 16, True, torch.float16),  # fewer tokens than rows: rows that see none
    ([130], 33, None, 4, 2, 128, 64, True, torch.float16),  # several row blocks
    ([4100], 1, None, 2, 2, 64, 128, False, torch.bfloat16),
    # more than 64 rows a key/value head
    ([600, 64, 0, 63], 17, [17, 17, 0, 5], 8, 2, 128, 16, True, torch.bfloat16),
    ([65, 1000], 33, None, 8, 2, 64, 32, False, torch.float16),
    ([300, 40], 40, None, 4, 1, 128, 64, True, torch.float16),  # two tiles, the second of 32 rows; fewer tokens than rows
    ([777], 129, None, 1, 1, 64, 256, True, torch.bfloat16),
    ([1, 2, 500], 10, None, 8, 1, 128, 128, False, torch.bfloat16),
    ([0, 0], 70, None, 1, 1, 64, 16, False, torch.float16),
    ([2100], 24, None, 6, 2, 128, 32, True, torch.float16),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"{c[0][0]}x{len(c[0])}-n{c[1]}-h{c[3]}.{c[4]}-d{c[5]}-p{c[6]}")
def test_attention_against_oracle(case):
    lens, n, new, H, HK, d, page, causal, dtype = case
    cache, table = filled(lens, HK, d, page, dtype, seed=sum(lens) + n)
    q = torch.randn(len(lens), n, H, d, generator=torch.Generator().manual_seed(n)).to(dtype)
    o, lse = check_attention(q, cache, table, lens, causal, new)
    for b in range(len(lens)):
        for i in range(n):
            if i >= (new[b] if new else n) or lens[b] == 0:
                assert not o[b, i].any() and torch.all(lse[b, :, i] == -math.inf)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
def test_random_shapes(d, dtype):
    g = torch.Generator().manual_seed(d + (dtype == torch.float16))  # up to 9 x 14 rows
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    for trial in range(12):
        B, n, HK = r(1, 5), r(1, 14), r(1, 4)
        H = HK * r(1, 9)
        lens = [r(0, 900) for _ in range(B)]
        new = [r(0, n) for _ in range(B)] if r(0, 1) else None
        page = 16 << r(0, 4)
        cache, table = filled(lens, HK, d, page, dtype, seed=trial)
        q = torch.randn(B, n, H, d, generator=g).to(dtype)
        check_attention(q, cache, table, lens, bool(r(0, 1)), new)


@pytest.mark.parametrize("n", [1, 6, 30])
def test_tables_wider_than_the_sequences(n):
    # the same sequences by tables of 512 tokens' capacity and more: items in one piece and in several
    lens, page = [512, 0, 301, 1, 128], 16
    cache, table = filled(lens, 3, 128, page, torch.bfloat16, seed=n)
    q = torch.randn(5, n, 6, 128, generator=torch.Generator().manual_seed(n)).bfloat16()
    assert table.shape[1] >= 32
    for width in (32, 33, 64, 200):
        wide = torch.full((5, width), -1, dtype=torch.int32)
        wide[:, :32] = table[:, :32]
        check_attention(q, cache, wide, lens, True)


@pytest.mark.parametrize("k_scale,v_scale,q_scale", [(8.0, 1.0, 3.0), (1e-3, 1e-4, 1.0), (1.0, 200.0, 30.0), (30.0, 1.0, 1e-3)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_ranges(dtype, k_scale, v_scale, q_scale):
    lens = [513, 70]
    cache, table = filled(lens, 2, 128, 32, dtype, seed=5, k_scale=k_scale, v_scale=v_scale)
    q = (torch.randn(2, 2, 4, 128, generator=torch.Generator().manual_seed(9)) * q_scale).to(dtype)
    check_attention(q, cache, table, lens, True)


@pytest.mark.parametrize("n", [1, 50])
def test_rising_maximum_and_steps(n):
    # scores and values' steps that grow along the sequence: the references move on every step
    lens, d, page = [640], 64, 64
    table, n_pages = pages(lens, page, 1)
    cache = noise_cache(n_pages, 1, page, d)
    g = torch.Generator().manual_seed(2)
    u = torch.randn(d, generator=g)
    t = torch.arange(640)
    k = (u * t[:, None] * 0.02 + 0.1 * torch.randn(640, d, generator=g)).half()
    v = (torch.randn(640, d, generator=g) * 2.0 ** (t[:, None] / 64.0 - 5)).half()
    for w, x in ((0, k), (1, v)):
        cache[table[0, t // page].long(), 0, w, t % page] = oc.pack_rows(*oc.quantise64(x, torch.float16), torch.float16)
    q = torch.stack([u, -u, 0 * u]).half().view(1, 1, 3, d).expand(1, n, 3, d) * torch.linspace(1, 0.1, n).half().view(1, n, 1, 1)
    check_attention(q, cache, table, lens, False)


def test_softmax_scale_and_lse_optional():
    cache, table = filled([100], 1, 64, 16, torch.float16)
    q = torch.randn(1, 1, 2, 64, generator=torch.Generator().manual_seed(1)).half()
    check_attention(q, cache, table, [100], False, scale=0.3)
    dev = (q.cuda(), cache.cuda(), table.cuda(), ints([100]).cuda())
    o, none = fa.forward_cache4(*dev)
    assert none is None and torch.equal(o, fa.forward_cache4(*dev, return_lse=True)[0])


@pytest.mark.parametrize("n", [4, 45])
def test_nan_in_masked_places_stays_there(n):
    # NaN keys and values behind a row's position must not reach it; a visible one must
    lens = [50]
    cache, table = filled(lens, 1, 128, 16, torch.float16, seed=3)
    q = torch.randn(1, n, 2, 128, generator=torch.Generator().manual_seed(1)).half()
    clean, _ = check_attention(q, cache, table, lens, True)
    for side in (0, 1):
        bad = cache.clone()
        bad[table[0, 48 // 16], 0, side, 48 % 16, 64:] = 255  # token 48: the last two rows see it
        o, _ = fa.forward_cache4(q.cuda(), bad.cuda(), table.cuda(), ints(lens).cuda(), None, True)
        fa.check_status(0)
        assert torch.equal(o[:, :-2].cpu().double(), clean[:, :-2])
        assert torch.isnan(o[:, -2:]).all()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("n", [2, 45])
def test_a_group_that_is_not_finite_leaves_the_other(n, value):
    # one visible token's step of the values' first 64 channels: those are lost, the others and lse are not
    lens = [300]
    cache, table = filled(lens, 1, 128, 16, torch.bfloat16, seed=n)
    q = torch.randn(1, n, 2, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    want, want_lse, weight, reach = oc.attention64(q, cache, table, lens)
    bad = cache.clone()
    bad[table[0, 100 // 16], 0, 1, 100 % 16, 64:66] = torch.tensor([value], dtype=torch.bfloat16).view(torch.uint8)
    o, lse = fa.forward_cache4(q.cuda(), bad.cuda(), table.cuda(), ints(lens).cuda(), return_lse=True)
    fa.check_status(0)
    o, lse = o.cpu().double(), lse.cpu().double()
    assert not torch.isfinite(o[..., :64]).any()
    tol = want.abs() * 2.0 ** -8 + (2.0 ** -11 + 2.0 ** -18 * reach[..., None] + 2.0 ** -15) * weight
    assert torch.all(((o - want).abs() <= tol)[..., 64:])
    assert torch.all((lse - want_lse).abs() <= 2.0 ** -19 * reach.transpose(1, 2) + 2.0 ** -15 + 2.0 ** -22 * want_lse.abs())


def test_negative_steps_are_taken_as_written():
    # the format allows any s; rows from elsewhere may hold negative ones
    cache, table = filled([40], 1, 64, 16, torch.float16, seed=6)
    c, s, m = oc.unpack_rows(cache, torch.float16)
    s = torch.where(torch.isfinite(s), s, torch.ones_like(s))
    m = torch.where(torch.isfinite(m), m, torch.ones_like(m))
    flipped = oc.pack_rows(15 - c, -s, m + 15 * s, torch.float16)
    q = torch.randn(1, 1, 1, 64, generator=torch.Generator().manual_seed(1)).half()
    _, fs, fm = oc.unpack_rows(oc.sequence_rows(flipped, table, 0, 40), torch.float16)
    want, want_lse, _, _ = oc.attention64(q, flipped, table, [40])
    o, lse = fa.forward_cache4(q.cuda(), flipped.cuda(), table.cuda(), ints([40]).cuda(), return_lse=True)
    # terms s c and m of either sign: their magnitudes bound both errors (as above)
    size = float((15 * fs.abs() + fm.abs()).max())
    reach = float(q.double().abs().sum()) * size / 8
    assert torch.all((o.cpu().double() - want).abs() <= want.abs() * 2.0 ** -11 + size * (2.0 ** -11 + 2.0 ** -18 * reach + 2.0 ** -15))
    assert abs(lse.item() - want_lse.item()) <= 2.0 ** -19 * reach + 2.0 ** -15 + 2.0 ** -22 * abs(want_lse.item())


# --- values whose steps lie far apart --------------------------------------------------------------------
def stepped(x, s, d, dtype, seed=0, low=-7.5):
    """(cache, table) of one sequence and head whose scores are exactly x[t] log2 units (ones_query) and whose values
    have steps of s[t] to 2 s[t] and minima of `low` steps; a step of 0 stands for the constant 1."""
    T, G = len(x), d // 64
    g = torch.Generator().manual_seed(seed)
    x = x.to(dtype).double()[:, None].expand(T, G)
    none = torch.zeros(T, G, dtype=torch.float64)
    s = s.double()[:, None] * (1 + torch.rand(T, G, generator=g).double())
    s = s.to(dtype).double()
    m = torch.where(s == 0, torch.ones_like(s), torch.where(torch.isfinite(s), low * s, none))
    codes = torch.randint(0, 16, (T, d), generator=g) * (s > 0).repeat_interleave(64, -1)
    table, n_pages = pages([T], 16, seed)
    cache, t = noise_cache(n_pages, 1, 16, d, seed), torch.arange(T)
    cache[table[0, t // 16].long(), 0, 0, t % 16] = oc.pack_rows(torch.zeros(T, d, dtype=torch.long), none, x, dtype)
    cache[table[0, t // 16].long(), 0, 1, t % 16] = oc.pack_rows(codes, s, m, dtype)
    return cache, table


def ones_query(n, d, dtype):
    # two heads; at scale ln 2 the first one's scores are the keys' constants, the second one's half of them
    return torch.tensor([1.0, 0.5])[:, None].expand(1, n, 2, d).to(dtype) / d


def check_steps(q, cache, table, T, causal, rows=None):
    """As check_attention, for steps of any size.  The rounded p s' multiplies a code with a mean taken off, which is 15
    at most in magnitude and which the other sum gives back: both sums' terms reach p (15 s' + |m'|).  Products far
    below a row's largest keep fewer bits: the largest stands at 2^7 or more of fp16, whose smallest step is 2^-24, so
    each is off by 2^-32 of it beside 2^-11 relative (in the kernel for many rows twice, where a reference moves within
    a step), times 15: T 2^-27.  The fp32 sums pass 15 times the largest and are rounded, towards zero even, twice in
    16 tokens: T 2^-22."""
    n = q.shape[1]
    rows = list(range(n)) if rows is None else rows
    o, lse = fa.forward_cache4(q.cuda(), cache.cuda(), table.cuda(), ints([T]).cuda(), None, causal, math.log(2), True)
    fa.check_status(0)
    o, lse = o.cpu().double(), lse.cpu().double()
    d, dtype = q.shape[3], q.dtype
    kr, vr = oc.sequence_rows(cache, table, 0, T)[:, :, 0]
    key = oc.unpack_rows(kr, dtype)[2][:, 0]
    codes, s, m = oc.unpack_rows(vr, dtype)
    for i in rows:
        see = T - n + i + 1 if causal else T
        for h in range(2):
            score = key[:see] * (1.0, 0.5)[h]  # log2 units
            p = torch.softmax(score * math.log(2), 0)
            step, low = s[:see].repeat_interleave(64, -1), m[:see].repeat_interleave(64, -1)
            want, weight = p @ (codes[:see] * step + low), p @ (15 * step + low.abs())
            largest = (p[:, None] * s[:see]).max()
            reach = float(score.abs().max()) * math.log(2)
            tol = want.abs() * torch.finfo(dtype).eps / 2 + (2.0 ** -11 + 2.0 ** -18 * reach + 2.0 ** -15) * weight + TINY[dtype]
            tol = tol + see * 2.0 ** -21 * largest
            err = (o[0, i, h] - want).abs()
            assert torch.all(err <= tol), f"row {i} head {h}: largest error over tolerance {(err / tol).max().item():.3g}"
            want = torch.logsumexp(score * math.log(2), 0).item()
            assert abs(lse[0, h, i].item() - want) <= 2.0 ** -19 * reach + 2.0 ** -15 + 2.0 ** -22 * abs(want)


def uneven(T, seed):
    return torch.rand(T, generator=torch.Generator().manual_seed(seed)) * 2 - 1


@pytest.mark.parametrize("d", [64, 128])
def test_a_maximum_that_jumps_between_the_halves_of_a_step(d):
    # 128 rows: tokens 32 on are 25 log2 units above those before, whose steps are 2^19 times theirs
    T = 64
    x, s = torch.zeros(T), torch.ones(T)
    x[32:] = 25
    s[:32] = 2.0 ** 19
    cache, table = stepped(x, s, d, torch.bfloat16, 1, low=0.0)
    check_steps(ones_query(64, d, torch.bfloat16), cache, table, T, False)


@pytest.mark.parametrize("dtype,ratio", [(torch.bfloat16, 2.0 ** 24), (torch.bfloat16, 2.0 ** 30), (torch.bfloat16, 2.0 ** 90),
                                         (torch.float16, 2.0 ** 28), (torch.bfloat16, math.inf)])
@pytest.mark.parametrize("n,d", [(4, 128), (8, 64), (45, 128), (45, 64), (33, 128)])
def test_large_steps_in_masked_places_stay_there(n, d, dtype, ratio):
    # the last three tokens' steps are out of all proportion; rows that do not see them keep every bit
    T = 50
    s = torch.full((T,), 2.0 ** -14 if dtype == torch.float16 else 1.0)
    s[-3:] *= ratio
    cache, table = stepped(uneven(T, n), s, d, dtype, 2)
    check_steps(ones_query(n, d, dtype), cache, table, T, True, rows=range(n - 3))


@pytest.mark.parametrize("gap,ratio", [(58, 2.0 ** 24), (58, 2.0 ** 40), (40, 2.0 ** 60), (100, 2.0 ** 95), (12, 2.0 ** 20)])
@pytest.mark.parametrize("n,d", [(1, 128), (3, 64), (45, 128), (45, 64), (33, 128)])
@pytest.mark.parametrize("T,at", [(100, 0), (100, 37), (3000, 5)])
def test_a_large_step_of_little_weight(T, at, n, d, gap, ratio):
    # one token's step is far above the others' and its score far below: what they lose is measured by its product
    x, s = uneven(T, n), torch.ones(T)
    x[at] = -gap
    s[at] = ratio
    cache, table = stepped(x, s, d, torch.bfloat16, 3)
    check_steps(ones_query(n, d, torch.bfloat16), cache, table, T, False)


@pytest.mark.parametrize("n,d", [(1, 128), (3, 64), (45, 128), (45, 64), (33, 128)])
@pytest.mark.parametrize("T,at", [(131, 130), (40, 39), (2000, 1999)])
def test_constant_values_before_a_large_step(T, at, n, d):
    # values without a step, then one of 2^100 and a weight of 2^-10: the first ones' weights stay in the sum
    x, s = torch.zeros(T), torch.zeros(T)
    x[at] = -10
    s[at] = 2.0 ** 100
    cache, table = stepped(x, s, d, torch.bfloat16, 4, low=0.0)
    check_steps(ones_query(n, d, torch.bfloat16), cache, table, T, False)


@pytest.mark.parametrize("n,d", [(2, 128), (40, 64)])
def test_steps_that_rise_and_fall(n, d):
    # products move over 2^80 along the sequence in both directions, the scores against them
    T = 1500
    t = torch.arange(T).double()
    s = 2.0 ** (40 * torch.sin(t / 90)).float()
    x = (30 * torch.cos(t / 50)).float()
    cache, table = stepped(x, s, d, torch.bfloat16, 5)
    check_steps(ones_query(n, d, torch.bfloat16), cache, table, T, True)


# --- lengths and pages that are wrong --------------------------------------------------------------------
@pytest.mark.parametrize("entry", ["write", "read", "attend", "attend many"])
@pytest.mark.parametrize("fault", ["page low", "page high", "length high", "length low", "new high", "new low"])
def test_bad_tables_and_lengths_are_reported(entry, fault):
    table, lens, new = ints([[0, 1], [2, 3]]), ints([20, 30]), ints([2, 2])
    if fault == "page low":
        table[1, 1] = -1
    elif fault == "page high":
        table[1, 1] = 4
    elif fault == "length high":
        lens[1] = 33
    elif fault == "length low":
        lens[1] = -1
    elif fault == "new high":
        new[1] = 3
    else:
        new[1] = -1
    cache = torch.zeros(4, 1, 2, 16, 36, dtype=torch.uint8, device="cuda")
    x = torch.ones(2, 2, 1, 64, dtype=torch.float16, device="cuda")
    table, lens, new = table.cuda(), lens.cuda(), new.cuda()
    fa.check_status(0)
    if entry == "write":
        fa.cache4_write(x, x, cache, table, lens, new)
    elif entry == "read":
        fa.cache4_read(cache, table, lens, 2, torch.float16, new)
    else:  # 2 or 128 query rows
        q = x if entry == "attend" else x.expand(2, 2, 64, 64)
        fa.forward_cache4(q, cache, table, lens, new_lens=new)
    torch.cuda.synchronize()
    want = "page_table" if fault.startswith("page") else "kv_lens"
    with pytest.raises(RuntimeError, match=f"earlier launch on cuda:0.*{want}"):
        fa.forward_cache4(x, cache, ints([[0, 1], [2, 3]]).cuda(), ints([20, 30]).cuda())
    fa.check_status(0)  # raised once
    if entry == "write":  # the other sequence's rows were written, no others
        used = cache.flatten(1).any(-1).tolist()
        assert used == [False, True, False, False]


@pytest.mark.parametrize("n", [3, 40])
def test_idle_sequences_need_no_pages(n):
    # a place of the batch without new rows keeps an old length, and its pages are gone
    cache, table = filled([200, 90], 2, 128, 16, torch.float16, seed=n)
    q = torch.randn(2, n, 4, 128, generator=torch.Generator().manual_seed(n)).half()
    idle, new = table.clone(), [n, 0]
    idle[1] = -1
    for causal in (False, True):
        o, lse = fa.forward_cache4(q.cuda(), cache.cuda(), idle.cuda(), ints([200, 90]).cuda(), None, causal, None, True, ints(new).cuda())
        fa.check_status(0)
        assert not o[1].any() and torch.all(lse[1] == -math.inf)
        check_attention(q, cache, table, [200, 90], causal, new, got=(o, lse))
    x = q[:, :, :2].cuda()
    fa.cache4_write(x, x, cache.cuda(), idle.cuda(), ints([200, 90]).cuda(), ints(new).cuda())
    k, v = fa.cache4_read(cache.cuda(), idle.cuda(), ints([200, 90]).cuda(), n, torch.float16, ints(new).cuda())
    fa.check_status(0)
    assert not k[1].any() and not v[1].any()


def test_new_rows_beyond_the_sequence_are_refused_by_the_movers():
    # a sequence shorter than the rows to write has no place for them; attention allows it (rows that see nothing)
    cache = torch.zeros(2, 1, 2, 16, 36, dtype=torch.uint8, device="cuda")
    x = torch.ones(1, 3, 1, 64, dtype=torch.float16, device="cuda")
    fa.cache4_write(x, x, cache, ints([[0]]).cuda(), ints([2]).cuda())
    with pytest.raises(RuntimeError, match="kv_lens"):
        fa.check_status(0)
    assert not cache.any()
    fa.forward_cache4(x, cache, ints([[0]]).cuda(), ints([2]).cuda())
    fa.check_status(0)


def test_refusals():
    cache = torch.zeros(4, 2, 2, 16, 36, dtype=torch.uint8, device="cuda")
    x = torch.zeros(2, 3, 2, 64, dtype=torch.float16, device="cuda")
    table, lens = ints([[0, 1], [2, 3]]).cuda(), ints([20, 30]).cuda()
    w = lambda **o: fa.cache4_write(**{**dict(k=x, v=x, cache=cache, page_table=table, kv_lens=lens), **o})
    r = lambda **o: fa.cache4_read(**{**dict(cache=cache, page_table=table, kv_lens=lens, n=3, dtype=torch.float16), **o})
    a = lambda **o: fa.forward_cache4(**{**dict(q=x, cache=cache, page_table=table, kv_lens=lens), **o})
    shared = [
        (dict(cache=cache.char()), "uint8"),
        (dict(cache=cache[..., :20]), "rows of"),
        (dict(cache=cache[:, :, :, :12]), "page_size"),
        (dict(cache=cache[:, :, :, ::2][:, :, :, :8]), "page_size"),
        (dict(cache=torch.zeros(4, 2, 2, 32, 36, dtype=torch.uint8, device="cuda")[:, :, :, ::2]), "dense"),
        (dict(cache=cache[:0]), "positive"),
        (dict(cache=cache[:1].expand(4, 2, 2, 16, 36)), "invalid argument"),
        (dict(page_table=table.long()), "int32"),
        (dict(page_table=table.t()), "contiguous rows"),
        (dict(page_table=table[0]), "page_table must be"),
        (dict(page_table=table.cpu()), "CUDA tensor"),
        (dict(kv_lens=lens.long()), "int32"),
        (dict(kv_lens=lens[:1]), "kv_lens must be"),
        (dict(kv_lens=ints([1, 2, 3, 4]).cuda()[::2]), "kv_lens must be"),
        (dict(new_lens=lens[:1]), "new_lens must be"),
        (dict(new_lens=lens.long()), "int32"),
    ]
    for fn in (w, r, a):
        for over, match in shared:
            with pytest.raises(RuntimeError, match=match):
                fn(**over)
    for over, match in [(dict(v=x[:1]), "same shape"), (dict(v=x.bfloat16()), "same data type"), (dict(k=x.float(), v=x.float()), "Only fp16"),
                        (dict(k=x[:, :, :1], v=x[:, :, :1]), "do not match"), (dict(k=x[..., :32], v=x[..., :32]), "do not match"),
                        (dict(k=x[:, :0], v=x[:, :0]), "positive"), (dict(k=x.transpose(2, 3)), "contiguous"), (dict(k=x.cpu()), "CUDA tensor")]:
        with pytest.raises(RuntimeError, match=match):
            w(**over)
    for over, match in [(dict(n=0), "n must be"), (dict(dtype=torch.float32), "Only fp16"), (dict(k_out=x[:, :2]), "k_out must be"),
                        (dict(v_out=x.bfloat16()), "v_out must be")]:
        with pytest.raises(RuntimeError, match=match):
            r(**over)
    for over, match in [(dict(q=x[:, :, :1]), "multiple of"), (dict(q=x.float()), "Only fp16"), (dict(q=x[..., :32].contiguous()), "differ"),
                        (dict(softmax_scale=0.0), "softmax_scale"), (dict(softmax_scale=1e-60), "fp32's range"),
                        (dict(softmax_scale=math.inf), "fp32's range"), (dict(softmax_scale=math.nan), "positive"), (dict(o=x[:1]), "same shape"), (dict(o=x.bfloat16()), "dtype")]:
        with pytest.raises(RuntimeError, match=match):
            a(**over)
    fa.check_status(0)


def test_what_autograd_follows_is_refused():
    # the three operators have no gradient: inputs and given outputs that ask for one are refused, not cut off
    import torch.autograd.forward_ad as fwd

    cache = torch.zeros(4, 2, 2, 16, 36, dtype=torch.uint8, device="cuda")
    x = torch.ones(2, 3, 2, 64, dtype=torch.float16, device="cuda")
    table, lens = ints([[0, 1], [2, 3]]).cuda(), ints([20, 30]).cuda()
    calls = [lambda t: fa.forward_cache4(t, cache, table, lens), lambda t: fa.forward_cache4(x, cache, table, lens, t),
             lambda t: fa.cache4_write(t, x, cache, table, lens), lambda t: fa.cache4_write(x, t, cache, table, lens),
             lambda t: fa.cache4_read(cache, table, lens, 3, torch.float16, None, t),
             lambda t: fa.cache4_read(cache, table, lens, 3, torch.float16, None, None, t)]
    trained = x.clone().requires_grad_()
    for call in calls:
        for t in (trained, trained * 2):
            with pytest.raises(RuntimeError, match="not differentiable"):
                call(t)
            if t.is_leaf:
                with torch.no_grad():
                    call(t)
        call(trained.detach().clone())
        with fwd.dual_level(), pytest.raises(RuntimeError, match="not differentiable"):
            call(fwd.make_dual(x.clone(), x))
    fa.check_status(0)


def test_wait_that_runs_out_is_reported():
    # nothing is loaded: the waits of the kernel for many rows run out, the context stays usable
    import ctypes

    from ampere_flash_attention_from_scratch_b200 import _abi

    lib = _abi.load()
    cache, table = filled([300, 70], 2, 128, 32, torch.float16, seed=11)
    q = torch.randn(2, 40, 4, 128, generator=torch.Generator().manual_seed(1)).half()
    qd, cd, td, ld = q.cuda(), cache.cuda(), table.cuda(), ints([300, 70]).cuda()
    o, lse = torch.zeros_like(qd), torch.zeros(2, 4, 40, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    c = _abi.AfaCache4()
    c.cache, c.page_stride, c.page_table, c.table_stride = cd.data_ptr(), cd.stride(0), td.data_ptr(), td.stride(0)
    c.kv_lens, c.status = ld.data_ptr(), status.data_ptr()
    c.n_pages, c.page_size, c.max_pages, c.batch, c.n_kv_heads, c.head_dim = cd.shape[0], 32, td.shape[1], 2, 2, 128
    c.dtype = _abi.AFA_DTYPE_FP16
    a = _abi.AfaCache4FwdArgs()
    bytes_ = lib.afa_cache4_fwd_workspace(ctypes.byref(c), 40, 4)
    ws = torch.empty(bytes_, dtype=torch.uint8, device="cuda")
    a.q, a.o, a.lse, a.workspace, a.workspace_bytes = qd.data_ptr(), o.data_ptr(), lse.data_ptr(), ws.data_ptr(), bytes_
    a.q_strides[:] = a.o_strides[:] = [qd.stride(0), qd.stride(1), qd.stride(2)]
    a.seq_len, a.n_heads, a.causal = 40, 4, 1
    stream = torch.cuda.current_stream().cuda_stream
    a.timeout_ns, a.test_flags = 20_000_000, _abi.AFA_TEST_PRODUCER_IDLE
    assert lib.afa_cache4_fwd_sm100(ctypes.byref(c), ctypes.byref(a), stream) == _abi.AFA_OK
    torch.cuda.synchronize()
    assert b"timeout: cache" in lib.afa_status_string(int(status.item()))
    status.zero_()
    a.timeout_ns, a.test_flags = 0, 0
    assert lib.afa_cache4_fwd_sm100(ctypes.byref(c), ctypes.byref(a), stream) == _abi.AFA_OK
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    check_attention(q, cache, table, [300, 70], True, got=(o, lse))


# --- streams, graphs, several calls ----------------------------------------------------------------------
@pytest.mark.parametrize("group", [4, 80])
def test_captured_steps_follow_their_inputs(group):
    # a decode step (write, attend) captured once and replayed as the sequences grow; two graphs side by side
    d, page, heads = 128, 16, 2
    graphs = []
    for i in range(2):
        table = torch.arange(8, dtype=torch.int32).view(2, 4).cuda()
        cache = torch.zeros(8, heads, 2, page, 72, dtype=torch.uint8, device="cuda")
        k, v = (torch.zeros(2, 1, heads, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        q = torch.zeros(2, 1, group * heads, d, dtype=torch.bfloat16, device="cuda")
        lens = ints([1, 1]).cuda()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            fa.cache4_write(k, v, cache, table, lens)
            fa.forward_cache4(q, cache, table, lens, return_lse=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            fa.cache4_write(k, v, cache, table, lens)
            o, lse = fa.forward_cache4(q, cache, table, lens, return_lse=True)
        graphs.append((graph, stream, k, v, q, lens, cache, table, o, lse))
    g = torch.Generator().manual_seed(1)
    for step in range(1, 60):
        for graph, stream, k, v, q, lens, *_ in graphs:
            for t in (k, v, q):
                t.copy_(torch.randn(t.shape, generator=g))
            lens.copy_(ints([step, max(1, step - 20)]))
        torch.cuda.synchronize()
        for graph, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        if step % 13 == 0:
            for _, _, k, v, q, lens, cache, table, o, lse in graphs:
                check_attention(q.cpu(), cache.cpu(), table.cpu(), lens.tolist(), False, got=(o, lse))
    fa.check_status(0)


@pytest.mark.parametrize("n", [1, 5, 40])
def test_capture_behind_copies_and_joined_streams(n):
    # calls whose predecessors in a graph are a copy, a fill, or the ends of two streams, and a call on a side stream
    d, page, B, HK = 128, 16, 2, 2
    g = torch.Generator().manual_seed(n)
    cache, table = filled([400, 70], HK, d, page, torch.bfloat16, seed=n)
    cache, table, lens = cache.cuda(), table.cuda(), ints([400, 70]).cuda()
    fresh = [torch.randn(B, n, 4 * HK, d, generator=g).bfloat16().cuda() for _ in range(3)]
    inv = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    pos = torch.zeros(1, B, n, dtype=torch.int32, device="cuda")
    x, q, o = (torch.zeros_like(fresh[0]) for _ in range(3))
    fill = torch.ones_like(x)

    def step(main, side):
        q.copy_(x)
        pos.fill_(7)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            turned, _ = fa.rotary(q, None, pos, inv)
            k = turned[:, :, :HK]
            fa.cache4_write(k, k, cache, table, lens)
        fill.zero_()
        main.wait_stream(side)
        fa.forward_cache4(turned, cache, table, lens, o, True)
        fill.add_(o)
        back, _ = fa.cache4_read(cache, table, lens, n, torch.bfloat16)
        return turned, back

    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(main):
        step(main, side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=main):
            turned, back = step(main, side)
        for f in fresh:
            x.copy_(f)
            graph.replay()
            torch.cuda.synchronize()
            want, _ = fa.rotary(f, None, pos, inv)
            assert torch.equal(turned, want) and torch.equal(fill, o)
            check_attention(want.cpu(), cache.cpu(), table.cpu(), [400, 70], True,
                            got=(o, fa.forward_cache4(want, cache, table, lens, None, True, None, True)[1]))
            assert torch.equal(back, fa.cache4_read(cache, table, lens, n, torch.bfloat16)[0])
    fa.check_status(0)


def test_inference_mode():
    # tensors without a version counter, as inputs, caches and given outputs
    table, lens = ints([[0, 1]]).cuda(), ints([20]).cuda()
    x = torch.randn(1, 20, 2, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    inv, pos = torch.ones(32, device="cuda"), torch.arange(20, device="cuda").view(1, 1, 20)

    def run():
        cache = fa.cache4_empty(2, 2, 16, 64)
        q, k = fa.rotary(x, x, pos, inv, q_out=torch.empty_like(x), k_out=torch.empty_like(x))
        fa.cache4_write(k, x, cache, table, lens)
        back = [torch.empty_like(x) for _ in range(2)]
        fa.cache4_read(cache, table, lens, 20, torch.float16, None, *back)
        o = torch.empty_like(x)
        fa.forward_cache4(q, cache, table, lens, o, True)
        return [q, k, *back, o]

    want = run()
    with torch.inference_mode():
        got = run()
    assert all(g.is_inference() and torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("n", [3, 40])
def test_calls_at_once_on_two_streams_agree_with_one(n):
    lens = [900, 1300, 5, 0]
    cache, table = filled(lens, 2, 128, 32, torch.float16, seed=4)
    cache, table, lens = cache.cuda(), table.cuda(), ints(lens).cuda()
    qs = [torch.randn(4, n, 8, 128, generator=torch.Generator().manual_seed(i)).half().cuda() for i in range(2)]
    want = [fa.forward_cache4(q, cache, table, lens, None, True, None, True) for q in qs]
    dense = torch.randn(1, 512, 4, 128, generator=torch.Generator().manual_seed(5)).half().cuda()
    want_dense, _ = fa.forward_ext(dense, dense, dense)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(20):
        got = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(fa.forward_cache4(q, cache, table, lens, None, True, None, True))
        between, _ = fa.forward_ext(dense, dense, dense)  # the dense kernel beside them
        torch.cuda.synchronize()
        assert torch.equal(between, want_dense)
        for a, b in zip(want, got):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        del got
    fa.check_status(0)


def test_result_does_not_depend_on_other_sequences_beyond_rounding():
    # the same sequence alone and in a ragged batch: the split differs, both hold to the oracle
    lens = [2000, 1, 777, 128, 3000, 64]
    cache, table = filled(lens, 1, 64, 64, torch.float16, seed=8)
    q = torch.randn(6, 1, 4, 64, generator=torch.Generator().manual_seed(2)).half()
    check_attention(q, cache, table, lens, False)
    check_attention(q[2:3], cache, table[2:3], lens[2:3], False)


@pytest.mark.parametrize("n", [1, 70])
def test_many_short_sequences(n):
    # more sequences than a warp has lanes, a few tokens each, one long among them
    lens = [(7 * b) % 37 for b in range(1100)]
    lens[700] = 900
    cache, table = filled(lens, 1, 64, 16, torch.float16, seed=9)
    q = torch.randn(1100, n, 1, 64, generator=torch.Generator().manual_seed(3)).half()
    dev = (q.cuda(), cache.cuda(), table.cuda(), ints(lens).cuda())
    o, lse = fa.forward_cache4(*dev, return_lse=True)
    some = [0, 1, 31, 32, 33, 699, 700, 701, 1098, 1099]
    check_attention(q[some], cache, table[some], [lens[b] for b in some], False, got=(o[some], lse[some]))
    kr, vr = fa.cache4_read(dev[1], dev[2], dev[3], 900, torch.float16, dev[3])
    fa.check_status(0)
    for b in some:
        rows = oc.sequence_rows(cache, table, b, lens[b])
        for got, r in ((kr, rows[0]), (vr, rows[1])):
            c, s, m = oc.unpack_rows(r, torch.float16)
            want = c * s.repeat_interleave(64, -1) + m.repeat_interleave(64, -1)
            assert torch.all((got[b, :lens[b]].cpu().double() - want).abs() <= 2.0 ** -11 * want.abs() * 1.001 + 2.0 ** -25)


def test_far_pages_pass_32_bit_offsets():
    # a pool of 5 GB: rows near its end are written, read and attended to
    n_pages = 5 * 2 ** 30 // (8 * 2 * 128 * 72)
    cache = torch.empty(n_pages, 8, 2, 128, 72, dtype=torch.uint8, device="cuda")
    assert cache.numel() > 2 ** 32
    table = ints([[n_pages - 1, n_pages - 2], [0, n_pages // 2]]).cuda()
    lens = ints([200, 200]).cuda()
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, 200, 8, 128, generator=g).half() for _ in range(2))
    fa.cache4_write(k.cuda(), v.cuda(), cache, table, lens)
    small = torch.stack([cache[i] for i in table.flatten().tolist()])
    near = ints([[0, 1], [2, 3]]).cuda()
    q = torch.randn(2, 1, 16, 128, generator=g).half()
    o, lse = fa.forward_cache4(q.cuda(), cache, table, lens, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(fa.cache4_read(cache, table, lens, 200, torch.float16),
                                                 fa.cache4_read(small, near, lens, 200, torch.float16)))
    check_attention(q, small.cpu(), near.cpu(), [200, 200], False, got=(o, lse))
    fa.check_status(0)


@pytest.mark.parametrize("case", [([1500, 700], 700, 8, 2, 128, 64, torch.bfloat16), ([900], 900, 4, 4, 64, 16, torch.float16)],
                         ids=lambda c: f"n{c[1]}-d{c[4]}")
def test_prompt_sized_chunks(case):
    # hundreds of new tokens at once, causal; the oracle's formulas on the GPU
    lens, n, H, HK, d, page, dtype = case
    new = [n, n - 300][: len(lens)]
    cache, table = filled(lens, HK, d, page, dtype, seed=12)
    q = torch.randn(len(lens), n, H, d, generator=torch.Generator().manual_seed(2)).to(dtype)
    o, lse = fa.forward_cache4(q.cuda(), cache.cuda(), table.cuda(), ints(lens).cuda(), None, True, None, True, ints(new).cuda())
    fa.check_status(0)
    for b, length in enumerate(lens):
        m = new[b]
        assert not o[b, m:].any() and torch.all(lse[b, :, m:] == -math.inf)
        part = []
        for r in oc.sequence_rows(cache, table, b, length):
            c, s, mn = oc.unpack_rows(r, dtype)
            part += [(c * s.repeat_interleave(64, -1)).cuda(), mn.repeat_interleave(64, -1).cuda()]
        kc, km, vc, vm = [x.transpose(0, 1).repeat_interleave(H // HK, 0) for x in part]  # [H, T, d]
        x = q[b, :m].cuda().double().transpose(0, 1)
        sees = torch.arange(length, device="cuda") <= length - m + torch.arange(m, device="cuda")[:, None]
        score = (x @ (kc + km).transpose(1, 2) / math.sqrt(d)).masked_fill(~sees, -math.inf)
        reach = (x.abs() @ (kc + km.abs()).transpose(1, 2) / math.sqrt(d)).masked_fill(~sees, 0).amax(-1)
        p = torch.softmax(score, -1)
        want, weight = p @ (vc + vm), p @ (vc + vm.abs())
        err = (o[b, :m].double().transpose(0, 1) - want).abs()
        eps = torch.finfo(dtype).eps
        tol = want.abs() * eps / 2 + (2.0 ** -11 + 2.0 ** -18 * reach[..., None] + 2.0 ** -15) * weight + TINY[dtype]
        assert torch.all(err <= tol), f"largest error over tolerance {(err / tol).max().item():.3f}"
        want_lse = torch.logsumexp(score, -1)
        assert torch.all((lse[b, :, :m].double() - want_lse).abs() <= 2.0 ** -19 * reach + 2.0 ** -15 + 2.0 ** -22 * want_lse.abs())


@pytest.mark.parametrize("capacity,n,HK", [(512, 1, 2), (2048, 2, 2), (4096, 24, 1)])
def test_calls_in_a_row_see_each_other(capacity, n, HK):
    # each call's inputs are the outputs of the one before, and the next one starts while that ends: the same as with
    # the device idle in between; narrow in one launch, in two, and the kernel for many rows
    d, page, H, B = 64, 16, 4 * HK, 3
    g = torch.Generator().manual_seed(capacity)
    first = torch.randn(B, n, H, d, generator=g).half().cuda()
    old = torch.randn(B, capacity, HK, d, generator=g).half().cuda()
    table = torch.randperm(B * capacity // page, generator=g).view(B, -1).int().cuda()
    inv = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().cuda()

    def run(idle):
        wait = torch.cuda.synchronize if idle else lambda: None
        cache = noise_cache(B * capacity // page, HK, page, d).cuda()
        fa.cache4_write(old, old, cache, table, ints([capacity] * B).cuda())
        lens = ints([capacity - 60 * n, 5, capacity // 2]).cuda()
        q, seen = first, []
        for _ in range(50):
            lens.add_(n)
            wait()
            pos = (lens[:, None] - n + torch.arange(n, device="cuda")).unsqueeze(0)
            q, k = fa.rotary(q, q[:, :, :HK], pos, inv, [32])
            wait()
            fa.cache4_write(k, q[:, :, HK:2 * HK], cache, table, lens)
            wait()
            o, _ = fa.forward_cache4(q, cache, table, lens, None, True)
            wait()
            back, _ = fa.cache4_read(cache, table, lens, n, torch.float16)
            wait()
            q = (o + back.repeat_interleave(4, 2)).clamp_(-4, 4)
            seen.append(q)
        torch.cuda.synchronize()
        return torch.stack(seen), cache

    want, got = run(True), run(False)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    assert torch.isfinite(got[0]).all() and got[0][-1].any()
    fa.check_status(0)


@pytest.mark.parametrize("n", [1, 300])
def test_rows_written_right_after_they_were_made(n):
    # one buffer of keys, turned anew by the kernel before each write: no write sees the buffer's last contents
    g = torch.Generator().manual_seed(n)
    src = [torch.randn(4, n, 8, 128, generator=g).half().cuda() for _ in range(4)]
    pos, inv = torch.arange(4 * n).view(1, 4, n).cuda(), torch.ones(64, device="cuda")
    table, n_pages = pages([n] * 4, 64)
    cache, table, lens = noise_cache(n_pages, 8, 64, 128).cuda(), table.cuda(), ints([n] * 4).cuda()
    k = torch.empty_like(src[0])
    want = []
    for x in src:
        fa.rotary(x, None, pos, inv, q_out=k)
        torch.cuda.synchronize()
        fa.cache4_write(k, k, cache, table, lens)
        want.append(fa.cache4_read(cache, table, lens, n, torch.float16)[0])
        torch.cuda.synchronize()
    got = []
    for i in range(100):
        fa.rotary(src[i % 4], None, pos, inv, q_out=k)
        fa.cache4_write(k, k, cache, table, lens)
        got.append(fa.cache4_read(cache, table, lens, n, torch.float16)[0])
    assert all(torch.equal(t, want[i % 4]) for i, t in enumerate(got))
    fa.check_status(0)


# --- together --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    """Positions, cache and attention as a model uses them: a ragged prompt is turned and written, attended to by
    forward_ext over the values read back, then tokens follow one and three at a time."""
    B, H, HK, d, page = 2, 8, 2, 128, 32
    prompt, g = [50, 81], torch.Generator().manual_seed(7)
    inv = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    table, n_pages = pages([200, 200], page, 3)
    cache = noise_cache(n_pages, HK, page, d).cuda()
    table = table.cuda()
    made = lambda n, h: torch.randn(B, n, h, d, generator=g).to(dtype).cuda()
    lens, n = list(prompt), max(prompt)
    q, k, v = made(n, H), made(n, HK), made(n, HK)
    pos = torch.arange(n).expand(3, B, n).cuda()
    q, k = fa.rotary(q, k, pos, inv, [16, 24, 24])
    fa.cache4_write(k, v, cache, table, ints(lens).cuda(), ints(lens).cuda())
    kr, vr = fa.cache4_read(cache, table, ints(lens).cuda(), n, dtype, ints(lens).cuda())
    for b in range(B):
        m = lens[b]
        dense, dense_lse = fa.forward_ext(q[b:b + 1, :m], kr[b:b + 1, :m], vr[b:b + 1, :m], None, True, None, True)
        o, lse = check_attention(q[b:b + 1, :m].cpu(), cache.cpu(), table[b:b + 1].cpu(), [m], True)
        # forward_ext sees K and V rounded to 16 bits and rounds P to them: its own parity bound against fp32
        tol = 1e-2 if dtype == torch.float16 else 4e-2
        assert (dense.cpu().double() - o).abs().max() <= tol
        assert (dense_lse.cpu().double() - lse).abs().max() <= tol
    for step in (1, 1, 3, 1):
        lens = [x + step for x in lens]
        q, k, v = made(step, H), made(step, HK), made(step, HK)
        pos = (ints(lens).cuda()[:, None] - step + torch.arange(step).cuda()).expand(3, B, step)
        q, k = fa.rotary(q, k, pos, inv, [16, 24, 24])
        fa.cache4_write(k, v, cache, table, ints(lens).cuda())
        got = fa.forward_cache4(q, cache, table, ints(lens).cuda(), None, True, None, True)
        check_attention(q.cpu(), cache.cpu(), table.cpu(), lens, True, got=got)
    fa.check_status(0)
