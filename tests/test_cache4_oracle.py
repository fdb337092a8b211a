"""The 64-bit oracles of the cache operators, pinned on the CPU, and the torch
entry points' refusal of host tensors."""

import math

import pytest
import torch

import afa_flash_attention_kernels as fa
from oracle import cache4_oracle as oc


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_float64_quantiser_equals_exact_arithmetic(dtype):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(40, 128, generator=g) * 2 + 1).to(dtype)
    x[3] = 1.5
    x[4, :64] = torch.arange(64) % 16
    for a, b in zip(oc.quantise64(x, dtype), oc.quantise_exact(x, dtype)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_round_fraction_is_the_types_own_rounding(dtype):
    from fractions import Fraction

    g = torch.Generator().manual_seed(2)
    for v in (torch.randn(200, generator=g) * 10.0 ** torch.randint(-7, 4, (200,), generator=g)).tolist():
        assert oc.round_fraction(Fraction(v), dtype) == torch.tensor(v, dtype=torch.float32).to(dtype).item()


def test_a_code_is_off_by_half_a_step():
    # |x - (s c + m)| <= s / 2 + the rounding of s times the code
    g = torch.Generator().manual_seed(3)
    x = torch.randn(50, 128, generator=g).to(torch.bfloat16)
    codes, s, m = oc.quantise64(x, torch.bfloat16)
    back = codes.double() * s.repeat_interleave(64, -1) + m.repeat_interleave(64, -1)
    half = s.repeat_interleave(64, -1) * (0.5 + 15 * 2.0 ** -8)
    assert torch.all((x.double() - back).abs() <= half)
    rows = oc.pack_rows(codes, s, m, torch.bfloat16)
    assert rows.shape[-1] == 72
    for a, b in zip(oc.unpack_rows(rows, torch.bfloat16), (codes, s, m)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("causal", [False, True])
def test_attention64_against_torch(causal):
    g = torch.Generator().manual_seed(4)
    B, N, H, HK, d, page = 2, 3, 4, 2, 64, 16
    lens = [37, 16]
    cache = torch.zeros(8, HK, 2, page, 36, dtype=torch.uint8)
    table = torch.tensor([[5, 0, 3], [7, -1, -1]])
    x = torch.randn(2, B, 48, HK, d, generator=g).half()
    for b, n in enumerate(lens):
        for t in range(n):
            for w in range(2):
                cache[table[b, t // page], :, w, t % page] = oc.pack_rows(*oc.quantise64(x[w, b, t], torch.float16), torch.float16)
    q = torch.randn(B, N, H, d, generator=g).half()
    o, lse, _, _ = oc.attention64(q, cache, table, lens, causal)
    for b, n in enumerate(lens):
        kv = []
        for w in range(2):
            c, s, m = oc.unpack_rows(oc.sequence_rows(cache, table, b, n)[w], torch.float16)
            kv.append((c * s.repeat_interleave(64, -1) + m.repeat_interleave(64, -1)).repeat_interleave(H // HK, 1).transpose(0, 1))
        mask = torch.ones(N, n, dtype=torch.bool).tril(n - N) if causal else None
        want = torch.nn.functional.scaled_dot_product_attention(q[b].double().transpose(0, 1), kv[0], kv[1], attn_mask=mask)
        assert torch.allclose(o[b], want.transpose(0, 1), atol=1e-12)
        score = q[b].double().transpose(0, 1) @ kv[0].transpose(1, 2) / math.sqrt(d)
        if causal:
            score = score.masked_fill(~mask, -math.inf)
        assert torch.allclose(lse[b], torch.logsumexp(score, -1), atol=1e-12)


def test_rotary64_against_complex_products():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 5, 3, 64, generator=g)
    pos = torch.randint(0, 1000, (2, 2, 5), generator=g)
    inv = torch.rand(16, generator=g)
    z = torch.polar(torch.ones(1, dtype=torch.float64), torch.cat([pos[0].double()[..., None] * inv[:4].double(),
                                                                   pos[1].double()[..., None] * inv[4:].double()], -1))
    z = z[:, :, None]
    got = oc.rotary64(x, pos, inv, [4, 12], True)
    want = torch.view_as_real(torch.view_as_complex(x.double()[..., :32].unflatten(-1, (16, 2)).contiguous()) * z).flatten(-2)
    assert torch.allclose(got[..., :32], want, atol=1e-13) and torch.equal(got[..., 32:], x[..., 32:].double())
    got = oc.rotary64(x, pos, inv, [4, 12], False)
    w = torch.complex(x.double()[..., :16], x.double()[..., 16:32]) * z
    assert torch.allclose(got[..., :32], torch.cat([w.real, w.imag], -1), atol=1e-13)
    back = oc.rotary64(got, pos, inv, [4, 12], False, inverse=True)
    assert torch.allclose(back, x.double(), atol=1e-13)


def test_entry_points_refuse_host_tensors():
    h = torch.zeros(2, 3, 4, 64, dtype=torch.float16)
    pos, inv = torch.zeros(1, 2, 3, dtype=torch.int64), torch.ones(32)
    cache = fa.cache4_empty(4, 4, 16, 64, torch.device("cpu"))
    assert cache.shape == (4, 4, 2, 16, 36) and cache.dtype == torch.uint8
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.full((2,), 3, dtype=torch.int32)
    for call in (lambda: fa.rotary(h, h, pos, inv), lambda: fa.cache4_write(h, h, cache, table, lens),
                 lambda: fa.cache4_read(cache, table, lens, 3, torch.float16), lambda: fa.forward_cache4(h, cache, table, lens)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()


@pytest.mark.parametrize("args,match", [((4, 4, 16, 96), "head_dim"), ((4, 4, 24, 64), "page_size"), ((0, 4, 16, 64), "positive"),
                                        ((4, -1, 16, 64), "positive")])
def test_cache4_empty_refusals(args, match):
    with pytest.raises(RuntimeError, match=match):
        fa.cache4_empty(*args, torch.device("cpu"))


@pytest.mark.parametrize("wrap", [2 ** 32, -2 ** 32, 2 ** 40])
def test_cache4_empty_head_dim_beyond_32_bits(wrap):
    with pytest.raises(RuntimeError, match="head_dim"):
        fa.cache4_empty(1, 1, 16, 64 + wrap, torch.device("cpu"))


def test_package_exports_the_operators():
    import ampere_flash_attention_from_scratch_b200 as pkg

    for name in ("rotary", "cache4_empty", "cache4_write", "cache4_read", "forward_cache4"):
        assert getattr(pkg, name) is getattr(fa, name)
