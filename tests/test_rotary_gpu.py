"""Rotary positions on the GPU against the 64-bit oracle.

Tolerance: one rounding of the result (half a step of its type, relative) plus, for the angle, sine, cosine and products in 32
bits, 2^-20 of the pair's magnitudes: the reduced angle is off by at most pi 2^-24 + 2^-32 turns, __sinf and __cosf by 2^-21 on
[-pi, pi], each product and sum by 2^-24."""

import pytest
import torch

from attn_engine import RotaryEmbedding
from core.native import lib
from oracle import paged_math as pm

pytestmark = pytest.mark.gpu


def draw(shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def check(got, x, want, rope, dtype):
    assert lib.last_device_status() == 0
    n = rope.rotary_dim // 2
    pair = torch.zeros_like(want)
    first = torch.arange(n) * 2 if rope.interleaved else torch.arange(n)
    second = first + (1 if rope.interleaved else n)
    both = (x[..., first].double().abs() + x[..., second].double().abs()) * rope.magnitude
    pair[..., first] = both
    pair[..., second] = both
    tol = want.abs() * (torch.finfo(dtype).eps / 2) + pair * 2.0 ** -20 + (2.0 ** -24 if dtype == torch.float16 else 0.0)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), (err - tol).max().item()
    assert torch.equal(got.cpu()[..., 2 * n:], x[..., 2 * n:].to(dtype))   # what does not turn stays as it is


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,part", [(64, 64), (128, 128), (128, 32), (192, 64), (80, 20), (6, 2), (256, 64), (40, 24)])
def test_types_layouts_and_parts(dtype, interleaved, D, part):
    B, S, H, Hkv = 2, 5, 6, 2
    rope = RotaryEmbedding(part, interleaved=interleaved)
    q, k = draw((B, S, H, D), dtype, 1), draw((B, S, Hkv, D), dtype, 2)
    pos = torch.tensor([[0, 1, 2, 3, 4], [1000000, 1000001, 7, -3, 2 ** 31 - 1]])
    a, b = rope(q.cuda(), k.cuda(), positions=pos.cuda())
    for got, x in ((a, q), (b, k)):
        check(got, x, pm.rotary(x, pos, rope.frequencies, 1.0, interleaved), rope, dtype)


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("yarn", 16.0)])
def test_stretched_frequencies(scaling, factor):
    rope = RotaryEmbedding(64, scaling=scaling, factor=factor)
    x, pos = draw((33, 3, 64), torch.float32, 3), torch.arange(33) * 30011
    check(rope(x.cuda(), positions=pos.cuda()), x, pm.rotary(x, pos, rope.frequencies, rope.magnitude), rope, torch.float32)


@pytest.mark.parametrize("how", ["default", "shared", "int32", "packed", "one_row", "expanded"])
def test_positions(how):
    B, S, H, D = 3, 7, 2, 64
    rope, x = RotaryEmbedding(D), draw((B, S, H, D), torch.float16, 4)
    pos = torch.arange(S).expand(B, S)
    given = None
    if how == "shared":
        pos = torch.arange(S).add(50).expand(B, S)
        given = pos[0].contiguous()
    elif how in ("int32", "packed"):
        pos = torch.arange(B * S).view(B, S) * 13
        given = pos.int()
    elif how == "one_row":
        pos = torch.arange(S).add(9).expand(B, S)
        given = pos[:1].contiguous()
    elif how == "expanded":
        pos = torch.tensor([[5], [6], [70000]]).expand(B, S)
        given = pos
    if how == "packed":
        got = rope(x.flatten(0, 1).cuda(), positions=given.flatten().cuda()).view(B, S, H, D)
    else:
        got = rope(x.cuda(), positions=None if given is None else given.cuda())
    check(got, x, pm.rotary(x, pos, rope.frequencies), rope, torch.float16)


def test_strided_heads_and_unaligned_rows():
    """Slices of wider heads, heads in front of tokens, and rows that begin anywhere (a value at a time)."""
    rope = RotaryEmbedding(64)
    for view in (lambda t: t[..., 64:128], lambda t: t.transpose(1, 2)[..., :64], lambda t: t[..., 3:67], lambda t: t[:, ::2, 1:, 8:72], lambda t: t[:1, :, :1, :64]):
        x = view(draw((2, 6, 4, 130), torch.bfloat16, 5))
        got = rope(view(draw((2, 6, 4, 130), torch.bfloat16, 5).cuda()))
        assert got.is_contiguous()
        check(got, x, pm.rotary(x, torch.arange(x.shape[1]).expand(x.shape[:2]), rope.frequencies), rope, torch.bfloat16)


def test_in_place_writes_the_view_and_nothing_else():
    rope = RotaryEmbedding(32)
    whole = draw((3, 4, 5, 96), torch.bfloat16, 6)
    dev = whole.cuda()
    with torch.no_grad():
        a = rope(dev[..., 32:80], inplace=True)
        rope(dev[:, :, :2, :32], inplace=True)
    assert a.data_ptr() == dev[..., 32:80].data_ptr()
    want = whole.double()
    pos = torch.arange(4).expand(3, 4)
    want[..., 32:80] = pm.rotary(whole[..., 32:80], pos, rope.frequencies)
    want[:, :, :2, :32] = pm.rotary(whole[:, :, :2, :32], pos, rope.frequencies)
    err = (dev.cpu().double() - want).abs()
    assert bool((err <= want.abs() * 2.0 ** -8 + 16 * 2.0 ** -20).all())
    same = torch.ones(96, dtype=torch.bool)
    same[:64] = False
    assert torch.equal(dev.cpu()[:, :, :, same], whole[:, :, :, same]) and torch.equal(dev.cpu()[:, :, 2:, :32], whole[:, :, 2:, :32])


def test_infinities_and_nans_stay_in_their_pair():
    rope, x = RotaryEmbedding(64), draw((4, 2, 64), torch.bfloat16, 7)
    clean = rope(x.cuda()).cpu()
    x[1, 0, 5], x[2, 1, 40] = float("nan"), float("inf")
    got = rope(x.cuda()).cpu()
    hit = torch.zeros(4, 2, 64, dtype=torch.bool)
    hit[1, 0, [5, 37]] = True
    hit[2, 1, [8, 40]] = True
    assert torch.equal(got[~hit], clean[~hit]) and bool(got[1, 0, [5, 37]].isnan().all()) and not bool(got[2, 1, [8, 40]].isfinite().any())


def test_many_heads_and_rows_share_their_angles():
    """More work than threads: heads are walked by a thread in turn."""
    rope = RotaryEmbedding(128)
    B, S, H = 2, 2100, 37
    q, k = draw((B, S, H, 128), torch.bfloat16, 8), draw((B, S, 3, 128), torch.bfloat16, 9)
    a, b = rope(q.cuda(), k.cuda())
    pos = torch.arange(S).expand(B, S)
    check(a, q, pm.rotary(q, pos, rope.frequencies), rope, torch.bfloat16)
    check(b, k, pm.rotary(k, pos, rope.frequencies), rope, torch.bfloat16)


def test_empty_operands():
    rope = RotaryEmbedding(64)
    q = torch.empty(2, 0, 4, 64, device="cuda", dtype=torch.bfloat16)
    assert rope(q).shape == q.shape
    q, k = torch.ones(2, 3, 4, 64, device="cuda", dtype=torch.bfloat16), torch.empty(2, 3, 0, 64, device="cuda", dtype=torch.bfloat16)
    a, b = rope(q, k)
    assert a.shape == q.shape and b.shape == k.shape


# ---------------------------------------------------------------------------------------------------------------
# gradients
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_are_the_rotation_back(dtype, interleaved):
    B, S, H, Hkv, D, part = 2, 6, 4, 2, 96, 64
    rope = RotaryEmbedding(part, interleaved=interleaved, scaling="yarn", factor=4.0)
    q, k = draw((B, S, H, D), dtype, 10).cuda().requires_grad_(), draw((B, S, Hkv, D), dtype, 11).cuda().requires_grad_()
    gq, gk = draw((B, S, H, D), dtype, 12), draw((B, S, Hkv, D), dtype, 13)
    pos = torch.arange(S).add(77777).expand(B, S)
    out = rope(q, k, positions=pos.cuda())
    dq, dk = torch.autograd.grad(out, (q, k), (gq.cuda(), gk.cuda()))
    for got, g in ((dq, gq), (dk, gk)):
        check(got, g, pm.rotary(g, pos, rope.frequencies, rope.magnitude, interleaved, -1.0), rope, dtype)


def test_gradient_against_differences():
    """The map is linear: the difference quotient is exact up to rounding, 2^-24 of values of order 1 over a step of 1."""
    rope = RotaryEmbedding(8)
    x, g, d = (draw((3, 2, 8), torch.float32, s).cuda() for s in (14, 15, 16))
    leaf = x.clone().requires_grad_()
    (grad,) = torch.autograd.grad(rope(leaf), leaf, g)
    quotient = ((rope(x + d) - rope(x - d)) * g).sum().item() / 2
    assert abs(quotient - (grad * d).sum().item()) <= 48 * 8 * 2.0 ** -20


def test_gradients_of_one_operand_broadcast_gradients_and_second_order():
    rope = RotaryEmbedding(16)
    q, k = draw((2, 3, 4, 16), torch.float32, 17).cuda(), draw((2, 3, 1, 16), torch.float32, 18).cuda().requires_grad_()
    a, b = rope(q, k)
    b.sum().backward()   # an expanded gradient
    pos = torch.arange(3).expand(2, 3)
    want = pm.rotary(torch.ones(2, 3, 1, 16), pos, rope.frequencies, 1.0, False, -1.0)
    assert (k.grad.cpu().double() - want).abs().max() <= 2.0 ** -18
    x = draw((3, 2, 16), torch.float32, 19).cuda().requires_grad_()
    (first,) = torch.autograd.grad((rope(x) ** 3).sum(), x, create_graph=True)
    (second,) = torch.autograd.grad(first.sum(), x)
    y = x.detach().cpu().double().requires_grad_()
    n, c = 8, torch.outer(torch.arange(3).double(), torch.tensor(rope.frequencies, dtype=torch.float64))
    co, si = c.cos().unsqueeze(1), c.sin().unsqueeze(1)
    z = torch.cat((y[..., :n] * co - y[..., n:] * si, y[..., n:] * co + y[..., :n] * si), -1)
    (f1,) = torch.autograd.grad((z ** 3).sum(), y, create_graph=True)
    (f2,) = torch.autograd.grad(f1.sum(), y)
    assert (second.cpu().double() - f2).abs().max() <= 1e-4 * f2.abs().max()


# ---------------------------------------------------------------------------------------------------------------
# refusals, streams, graphs
# ---------------------------------------------------------------------------------------------------------------

def test_refusals():
    rope = RotaryEmbedding(64)
    q = torch.zeros(2, 3, 4, 64, device="cuda", dtype=torch.bfloat16)
    for bad in (dict(q=q.double()), dict(q=q[0, 0]), dict(q=q[..., :32]), dict(q=q, k=q[:, :2]), dict(q=q, k=q.half()), dict(q=q.transpose(2, 3)),
                dict(q=q, positions=torch.arange(4, device="cuda")), dict(q=q, positions=torch.arange(3)), dict(q=q, positions=torch.arange(3., device="cuda")),
                dict(q=q.clone().requires_grad_(), inplace=True), dict(q=q[:, :, :1].expand(2, 3, 4, 64), inplace=True)):
        with pytest.raises(ValueError):
            rope(**bad)
    with pytest.raises(lib.NativeError):
        rope(q.cpu())


def test_other_stream_and_captured_replay():
    rope = RotaryEmbedding(64)
    x = draw((40, 4, 64), torch.bfloat16, 20)
    buf, pos = x.cuda(), torch.arange(40).cuda()
    want = rope(buf, positions=pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rope(buf, positions=pos)
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rope(buf, positions=pos)
    pos.add_(1000)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, rope(buf, positions=pos)) and not torch.equal(out, want)
    fresh = RotaryEmbedding(64)
    with pytest.raises(lib.NativeError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh(buf)


def test_captured_training_step():
    """Forward and backward in one graph, replayed with other inputs, positions and gradients."""
    rope = RotaryEmbedding(64)
    q, k = (draw((2, 33, h, 64), torch.bfloat16, 30 + h).cuda().requires_grad_() for h in (4, 2))
    gq, gk = (draw((2, 33, h, 64), torch.bfloat16, 40 + h).cuda() for h in (4, 2))
    pos = torch.arange(33).cuda()

    def step():
        yq, yk = rope(q, k, pos)
        return (yq.detach(), yk.detach(), *torch.autograd.grad((yq, yk), (q, k), (gq, gk)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (50, 60):
        with torch.no_grad():
            for i, t in enumerate((q, k, gq, gk)):
                t.copy_(draw(tuple(t.shape), torch.bfloat16, seed + i).cuda())
            pos.add_(777)
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
