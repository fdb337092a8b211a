"""Rotary positions on the GPU against the 64-bit oracle, and their gradients.

Tolerance: a turned value is rounded once to 16 bits (half a step, eps / 2
relative, or half of the smallest subnormal), from fp32 products whose operands
cos and sin are off by a few units in the 24th bit and whose angle is off by one
rounding of at most half a turn (2^-24 * pi): together below 2^-20 (|a| + |b|).
"""

import math

import pytest
import torch

import afa_flash_attention_kernels as fa
from oracle import cache4_oracle as oc

pytestmark = pytest.mark.gpu

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def _check(got, x, want, rot, interleaved):
    xd = x.double().cpu()
    size = xd.abs().clone()
    a = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    b = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    both = xd[..., a].abs() + xd[..., b].abs()
    size[..., a] = size[..., b] = both
    dt = got.dtype
    tol = want.abs() * (torch.finfo(dt).eps / 2) + size * 2.0 ** -20 + TINY[dt]
    err = (got.double().cpu() - want).abs()
    assert torch.all(err <= tol), f"largest error over tolerance {(err / tol).max().item():.3f}"
    assert torch.equal(got[..., rot:], x[..., rot:])


def _inv(pairs, base=10000.0):
    return (base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float()


CASES = [
    # B, N, H, HK, d, rot, sections, interleaved, dtype, far
    (1, 1, 1, 1, 128, 128, [64], False, torch.bfloat16, 1),
    (64, 1, 32, 8, 128, 128, [16, 24, 24], False, torch.bfloat16, 10 ** 6),
    (2, 333, 5, 1, 64, 64, [8, 12, 12], True, torch.float16, 500),
    (3, 77, 7, 7, 128, 64, [16, 16], False, torch.float16, 2 ** 31 - 1),
    (2, 50, 3, 2, 128, 16, [0, 8], True, torch.bfloat16, 100),
    (1, 9, 2, 3, 16, 16, [8], False, torch.float16, 100),
    (1, 13, 3, 1, 80, 48, [4, 20], True, torch.bfloat16, 4000),
    (1, 5, 2, 2, 512, 512, [32] * 8, False, torch.float16, 70000),
    (2, 2050, 4, 4, 64, 32, [16], False, torch.bfloat16, 131072),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:6])))
@pytest.mark.parametrize("kind", ["int64", "int32", "float32"])
def test_against_oracle(case, kind):
    B, N, H, HK, d, rot, sections, inter, dtype, far = case
    g = torch.Generator().manual_seed(N + d)
    q, k = (torch.randn(B, N, h, d, generator=g).to(dtype) for h in (H, HK))
    pos = torch.randint(0, far + 1, (len(sections), B, N), generator=g)
    pos = pos.to(getattr(torch, kind)) if kind != "float32" else (pos.double() * 0.37).float()
    inv = _inv(rot // 2)
    a, b = fa.rotary(q.cuda(), k.cuda(), pos.cuda(), inv.cuda(), sections, inter)
    for got, x in ((a, q), (b, k)):
        assert got.dtype == dtype and got.is_contiguous()
        _check(got.cpu(), x, oc.rotary64(x, pos, inv, sections, inter), rot, inter)
    c, none = fa.rotary(q.cuda(), None, pos.cuda(), inv.cuda(), sections, inter)
    assert none is None and torch.equal(c, a)


def test_negative_positions_and_inverse():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 9, 3, 64, generator=g).half()
    pos = torch.randint(-10 ** 6, 0, (1, 2, 9), generator=g)
    inv = _inv(32)
    a, _ = fa.rotary(q.cuda(), None, pos.cuda(), inv.cuda(), inverse=True)
    _check(a.cpu(), q, oc.rotary64(q, pos, inv, [32], False, inverse=True), 64, False)
    b, _ = fa.rotary(q.cuda(), None, -pos.cuda(), inv.cuda())
    assert torch.equal(a, b)


def test_strided_views_and_broadcasts():
    # q and k as slices of one packed projection, head-major storage, positions and inputs that repeat
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(2, 40, 3, 4, 128, generator=g).to(torch.bfloat16).cuda()
    pos = torch.arange(40).cuda().view(1, 1, 40).expand(3, 2, 40)
    inv = _inv(64).cuda()
    want = fa.rotary(qkv[:, :, 0].contiguous(), qkv[:, :, 1].contiguous(), pos.contiguous(), inv, [16, 24, 24])
    got = fa.rotary(qkv[:, :, 0], qkv[:, :, 1], pos, inv, [16, 24, 24])
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    hm = qkv[:, :, 0].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(fa.rotary(hm, None, pos, inv, [16, 24, 24])[0], want[0])
    rep = qkv[:1, :, 0].expand(2, 40, 4, 128)
    assert torch.equal(fa.rotary(rep, None, pos, inv, [16, 24, 24])[0][1], want[0][0])
    # outputs given: in place within the packed projection, the values between untouched
    keep = qkv.clone()
    q_out, k_out = qkv[:, :, 0], qkv[:, :, 1]
    a, b = fa.rotary(q_out, k_out, pos, inv, [16, 24, 24], q_out=q_out, k_out=k_out)
    assert a.data_ptr() == q_out.data_ptr() and torch.equal(a, want[0]) and torch.equal(b, want[1])
    assert torch.equal(qkv[:, :, 2], keep[:, :, 2])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients(dtype, inter):
    g = torch.Generator().manual_seed(3)
    q, k, dq, dk = (torch.randn(2, 31, h, 64, generator=g).to(dtype) for h in (4, 2, 4, 2))
    pos = torch.randint(0, 5000, (2, 2, 31), generator=g)
    inv = _inv(24)
    x, y = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    a, b = fa.rotary(x, y, pos.cuda(), inv.cuda(), [10, 14], inter)
    gx, gy = torch.autograd.grad((a, b), (x, y), (dq.cuda(), dk.cuda()))
    for got, up in ((gx, dq), (gy, dk)):
        _check(got.cpu(), up, oc.rotary64(up, pos, inv, [10, 14], inter, inverse=True), 48, inter)
    # one output's gradient only, one input's only, and upstream gradients that autograd expands
    a, b = fa.rotary(x, y, pos.cuda(), inv.cuda(), [10, 14], inter)
    (only,) = torch.autograd.grad(b, y, dk.cuda())
    assert torch.equal(only, gy)
    a, _ = fa.rotary(x, y.detach(), pos.cuda(), inv.cuda(), [10, 14], inter)
    a.sum().backward()
    ones = torch.ones_like(q)
    _check(x.grad.cpu(), ones, oc.rotary64(ones, pos, inv, [10, 14], inter, inverse=True), 48, inter)
    # the gradient is linear in the upstream one, with the forward as its own derivative
    up = dq.cuda().requires_grad_()
    a, _ = fa.rotary(x, None, pos.cuda(), inv.cuda(), [10, 14], inter)
    (gx2,) = torch.autograd.grad(a, x, up, create_graph=True)
    (back,) = torch.autograd.grad(gx2, up, q.cuda())
    assert torch.equal(gx2.detach(), gx) and torch.equal(back, a.detach())


def test_gradient_against_differences():
    # central differences of L = sum(w * rotary(q)) in float64 through the oracle; L is linear in q, so the
    # only error is the gradient's own rounding to bf16 and fp32
    g = torch.Generator().manual_seed(4)
    q, w = (torch.randn(1, 3, 1, 16, generator=g).to(torch.bfloat16) for _ in range(2))
    pos, inv = torch.tensor([[[3, 50, 700]]]), _inv(8)
    x = q.cuda().requires_grad_()
    (got,) = torch.autograd.grad(fa.rotary(x, None, pos.cuda(), inv.cuda())[0], x, w.cuda())
    for n in range(3):
        for c in range(16):
            hi, lo = q.double().clone(), q.double().clone()
            hi[0, n, 0, c] += 1
            lo[0, n, 0, c] -= 1
            L = [(w.double() * oc.rotary64(z, pos, inv, [8], False)).sum().item() for z in (hi, lo)]
            want = (L[0] - L[1]) / 2
            assert abs(got[0, n, 0, c].item() - want) <= abs(want) * 2.0 ** -8 + 2.0 ** -18


def test_gradient_of_shared_and_broadcast_inputs():
    # one tensor used as q and as k, and a key broadcast over the batch: gradients add up
    g = torch.Generator().manual_seed(5)
    q, d1, d2 = (torch.randn(2, 8, 2, 64, generator=g).half().cuda() for _ in range(3))
    pos, inv = torch.arange(16).view(1, 2, 8).cuda(), _inv(32).cuda()
    x = q.clone().requires_grad_()
    a, b = fa.rotary(x, x, pos, inv)
    (both,) = torch.autograd.grad((a, b), x, (d1, d2))
    one, two = fa.rotary(d1, d2, pos, inv, inverse=True)
    assert torch.equal(both, one + two)
    y = q[:1].clone().requires_grad_()
    a, _ = fa.rotary(y.expand(2, 8, 2, 64), None, pos, inv)
    (gy,) = torch.autograd.grad(a, y, d1)
    assert torch.equal(gy, one.sum(0, keepdim=True))


@pytest.mark.parametrize("trained", ["q", "k"])
def test_an_output_requires_a_gradient_if_its_input_does(trained):
    g = torch.Generator().manual_seed(7)
    q, k, up = (torch.randn(2, 6, 3, 64, generator=g).half().cuda() for _ in range(3))
    pos, inv = torch.arange(12).view(1, 2, 6).cuda(), _inv(32).cuda()
    x = (q if trained == "q" else k).requires_grad_()
    out = fa.rotary(q, k, pos, inv)
    ours, other = out if trained == "q" else out[::-1]
    assert ours.requires_grad and not other.requires_grad and other.grad_fn is None
    (gx,) = torch.autograd.grad(ours, x, up)
    assert torch.equal(gx, fa.rotary(up, None, pos, inv, inverse=True)[0])
    plain = fa.rotary(q.detach(), k.detach(), pos, inv)
    assert torch.equal(out[0], plain[0]) and torch.equal(out[1], plain[1])


def test_tangents():
    # forward mode: each output's tangent is its input's, turned; with one, the other or both, and through a graph
    import torch.autograd.forward_ad as fwd

    g = torch.Generator().manual_seed(8)
    q, k, dq, dk, up = (torch.randn(2, 6, 3, 64, generator=g).half().cuda() for _ in range(5))
    pos, inv = torch.arange(24).view(2, 2, 6).cuda(), _inv(24).cuda()
    turn = lambda x: fa.rotary(x, None, pos, inv, [10, 14], True)[0]
    tangent = lambda x: fwd.unpack_dual(x).tangent
    with fwd.dual_level():
        a, b = fa.rotary(fwd.make_dual(q, dq), fwd.make_dual(k, dk), pos, inv, [10, 14], True)
        assert torch.equal(tangent(a), turn(dq)) and torch.equal(tangent(b), turn(dk))
        assert torch.equal(fwd.unpack_dual(a).primal, turn(q)) and torch.equal(fwd.unpack_dual(b).primal, turn(k))
        a, b = fa.rotary(fwd.make_dual(q, dq), k, pos, inv, [10, 14], True)
        assert torch.equal(tangent(a), turn(dq)) and tangent(b) is None
        a, b = fa.rotary(q, fwd.make_dual(k, dk), pos, inv, [10, 14], True)
        assert tangent(a) is None and torch.equal(tangent(b), turn(dk))
        with torch.no_grad():  # which is about the other mode
            assert torch.equal(tangent(turn(fwd.make_dual(q, dq))), turn(dq))
        # a tangent that repeats, and one of zeros without memory
        assert torch.equal(tangent(turn(fwd.make_dual(q, dq[:1, :1].expand_as(q)))), turn(dq[:1, :1].expand_as(q).contiguous()))
        assert not tangent(turn(fwd.make_dual(q, torch._efficientzerotensor(q.shape, dtype=q.dtype, device="cuda")))).any()
        # in both modes at once: gradients of the output and of its tangent
        x, t = q.clone().requires_grad_(), dq.clone().requires_grad_()
        a = turn(fwd.make_dual(x, t))
        assert torch.equal(torch.autograd.grad(a, x, up, retain_graph=True)[0], fa.rotary(up, None, pos, inv, [10, 14], True, True)[0])
        assert torch.equal(torch.autograd.grad(tangent(a), t, up)[0], fa.rotary(up, None, pos, inv, [10, 14], True, True)[0])
        # and through the gradient: the tangent of a gradient is the upstream gradient's, turned back
        gx = torch.autograd.grad(turn(x), x, fwd.make_dual(up, dk), create_graph=True)[0]
        assert torch.equal(tangent(gx), fa.rotary(dk, None, pos, inv, [10, 14], True, True)[0])
        for kwargs in (dict(q_out=torch.empty_like(q)), dict(inv_freq=fwd.make_dual(inv, inv))):
            with pytest.raises(RuntimeError, match="tangent|not differentiable"):
                fa.rotary(**{**dict(q=fwd.make_dual(q, dq), k=None, positions=pos, inv_freq=inv, sections=[10, 14]), **kwargs})
        with pytest.raises(RuntimeError, match="must not"):
            fa.rotary(q, None, pos, inv, [10, 14], q_out=fwd.make_dual(q.clone(), dq))
    # linear: differences along the tangent in 64 bits
    want = oc.rotary64(dq.cpu(), pos.cpu(), inv.cpu(), [10, 14], True)
    diff = oc.rotary64((q.double() + dq.double()).cpu(), pos.cpu(), inv.cpu(), [10, 14], True) - oc.rotary64(q.cpu(), pos.cpu(), inv.cpu(), [10, 14], True)
    assert torch.allclose(want, diff, atol=1e-12)
    _check(turn(dq).cpu(), dq.cpu(), want, 48, True)


def test_capture_of_forward_and_backward():
    g = torch.Generator().manual_seed(6)
    q, dq = (torch.randn(2, 100, 4, 128, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    pos, inv = torch.arange(200).view(1, 2, 100).cuda(), _inv(64).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x = q.clone().requires_grad_()
        for _ in range(2):
            torch.autograd.grad(fa.rotary(x, None, pos, inv)[0], x, dq)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        a, _ = fa.rotary(x, None, pos, inv)
        (gx,) = torch.autograd.grad(a, x, dq)
    with torch.no_grad():
        x.copy_(q * 2)
        dq.mul_(2)
        pos.add_(7)
    graph.replay()
    torch.cuda.synchronize()
    with torch.no_grad():
        assert torch.equal(a, fa.rotary(x.detach(), None, pos, inv)[0])
        assert torch.equal(gx, fa.rotary(dq, None, pos, inv, inverse=True)[0])


def test_a_given_output_counts_as_written():
    # autograd refuses a backward pass through a tensor that was turned in place after it was saved
    q = torch.ones(1, 2, 1, 64, dtype=torch.float16, device="cuda")
    w = torch.ones_like(q).requires_grad_()
    y = (q * w).sum()
    pos, inv = torch.tensor([[[1, 2]]]).cuda(), _inv(32).cuda()
    fa.rotary(q, None, pos, inv, q_out=q)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        a, b = fa.rotary(q.clone(), q.clone(), pos, inv)
        assert torch.equal(a, b)


def test_many_heads_and_one():
    q = torch.randn(1, 2, 3000, 16, generator=torch.Generator().manual_seed(8)).half().cuda()
    pos, inv = torch.tensor([[[5, 900]]]).cuda(), _inv(8).cuda()
    a, _ = fa.rotary(q, None, pos, inv)
    for h in (0, 1499, 2999):
        assert torch.equal(a[:, :, h:h + 1], fa.rotary(q[:, :, h:h + 1], None, pos, inv)[0])
    with pytest.raises(RuntimeError, match="heads together"):
        fa.rotary(q.expand(1, 2, 3000, 16).repeat(1, 1, 3, 1), None, pos, inv)


def test_non_finite_values_stay_in_their_pair():
    q = torch.ones(1, 2, 1, 64, dtype=torch.float16)
    q[0, 0, 0, 3] = math.inf
    q[0, 1, 0, 40] = math.nan
    a, _ = fa.rotary(q.cuda(), None, torch.tensor([[[1, 2]]]).cuda(), _inv(32).cuda())
    bad = ~torch.isfinite(a.cpu())
    assert bad.nonzero().tolist() == [[0, 0, 0, 3], [0, 0, 0, 35], [0, 1, 0, 8], [0, 1, 0, 40]]


def test_refusals():
    q = torch.zeros(2, 3, 4, 64, dtype=torch.float16, device="cuda")
    pos, inv = torch.zeros(1, 2, 3, dtype=torch.int64, device="cuda"), torch.ones(32, device="cuda")
    bad = [
        ((q.float(), None, pos, inv), "Only fp16 and bf16"),
        ((q, q.bfloat16(), pos, inv), "same data type"),
        ((q, q[..., :32].contiguous(), pos, inv), "head_dim differ"),
        ((q, None, pos[:, :1], inv), "positions must be"),
        ((q, None, pos.double(), inv), "int32, int64 or float32"),
        ((q, None, pos, inv.double()), "inv_freq"),
        ((q, None, pos, torch.ones(40, device="cuda")), "inv_freq must hold"),
        ((q, None, pos, torch.ones(12, device="cuda")), "inv_freq must hold"),
        ((q, None, pos, inv, [16]), "add up"),
        ((q, None, pos, inv, [48, -16]), "one entry"),
        ((q, None, pos.expand(2, 2, 3), inv, [48, -16]), "negative"),
        ((q, None, pos.expand(2, 2, 3), inv), "one entry"),
        ((q.transpose(2, 3), None, pos, inv), "contiguous head_dim"),
        ((q[:0], None, pos[:, :0], inv), "positive"),
        ((q.cpu(), None, pos, inv), "must be a CUDA tensor"),
        ((q, None, pos.cpu(), inv), "same device"),
        ((q.view(-1)[4:-60].view(-1)[: 64 * 4].view(1, 1, 4, 64), None, pos[:, :1, :1], inv), "16-byte aligned"),
    ]
    for args, match in bad:
        with pytest.raises(RuntimeError, match=match):
            fa.rotary(*args)
    x = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="cannot be given"):
        fa.rotary(x, None, pos, inv, q_out=torch.empty_like(q))
    with pytest.raises(RuntimeError, match="not differentiable"):
        fa.rotary(q, None, pos, inv.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="same shape"):
        fa.rotary(q, None, pos, inv, q_out=q[:1])
    with pytest.raises(RuntimeError, match="k_out without k"):
        fa.rotary(q, None, pos, inv, k_out=q)
