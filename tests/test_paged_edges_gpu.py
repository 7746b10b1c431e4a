"""Calls of rotary positions and of paged caches at the edges of what they take: operands without heads, gradients that nobody
asked for, frequencies that leave while they are read, batches whose first rows go backwards, broadcast queries, pools that moved.
Tolerances are those of test_rotary_gpu.py and test_paged_gpu.py."""

import gc

import pytest
import torch

from attn_engine import PagedKVCache, RotaryEmbedding
from core.native import lib
from oracle import paged_math as pm

pytestmark = pytest.mark.gpu


def draw(shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---------------------------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_queries_without_heads_leave_the_keys_their_rotation(packed, dtype):
    """q [.., 0, D] beside k with heads: k turns as it does alone, forward, in place and backward."""
    rope, lead = RotaryEmbedding(64), (7,) if packed else (2, 7)
    q = torch.empty(*lead, 0, 64, dtype=dtype, device="cuda")
    k, g = draw((*lead, 3, 64), dtype, 1).cuda(), draw((*lead, 3, 64), dtype, 2).cuda()
    pos = torch.arange(7, device="cuda") + 500
    want = rope(k, positions=pos)
    a, b = rope(q, k, positions=pos)
    assert a.shape == q.shape and torch.equal(b, want)
    own = k.clone()
    with torch.no_grad():
        a, b = rope(q, own, positions=pos, inplace=True)
    assert b.data_ptr() == own.data_ptr() and torch.equal(own, want)
    leaf, empty = k.clone().requires_grad_(), q.clone().requires_grad_()
    (alone,) = torch.autograd.grad(rope(leaf, positions=pos), leaf, g)
    a, b = rope(empty, leaf, positions=pos)
    dq, dk = torch.autograd.grad((a, b), (empty, leaf), (torch.empty_like(a), g))
    assert dq.shape == q.shape and torch.equal(dk, alone)
    assert lib.last_device_status() == 0


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("both", [False, True])
def test_only_what_asks_for_a_gradient_gets_one(given, both):
    """An operand that wants none comes back without a graph (and may be appended); of two, each gradient is had by itself."""
    rope = RotaryEmbedding(64)
    pos = torch.arange(5, device="cuda") + 90 if given else None
    x, gx = draw((2, 5, 4, 64), torch.bfloat16, 5).cuda(), draw((2, 5, 4, 64), torch.bfloat16, 6).cuda()
    y, gy = draw((2, 5, 2, 64), torch.bfloat16, 7).cuda(), draw((2, 5, 2, 64), torch.bfloat16, 8).cuda()
    alone = []
    for t, g in ((x, gx), (y, gy)):
        leaf = t.clone().requires_grad_()
        alone += torch.autograd.grad(rope(leaf, positions=pos), leaf, g)
    for which in (0, 1):
        q, k = x.clone().requires_grad_(both or which == 0), y.clone().requires_grad_(both or which == 1)
        a, b = rope(q, k, positions=pos)
        assert a.requires_grad == q.requires_grad and b.requires_grad == k.requires_grad
        outputs, grads = ((a, b), (gx, gy)) if both else ((a, b)[which], (gx, gy)[which])
        (d,) = torch.autograd.grad(outputs, (q, k)[which], grads, retain_graph=True)
        assert torch.equal(d, alone[which])
        (again,) = torch.autograd.grad((a, b)[which], (q, k)[which], (gx, gy)[which], create_graph=True)
        assert torch.equal(again, alone[which])
        if not both and which == 0:
            cache = PagedKVCache.allocate(2, 16, 2, 64)
            table, lens = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda"), torch.tensor([5, 5], dtype=torch.int32, device="cuda")
            cache.append(b, b, table, lens)
            assert torch.equal(cache.read(table, lens, 5)[0], b)


def test_tensors_without_memory_are_refused():
    """Before anything is launched; a gradient of zeros that has none is zeros."""
    cache, table, lens = filled([30, 20], 2, 64, 16, torch.bfloat16, False, 9)

    def freed(*shape, dtype=torch.bfloat16):
        t = torch.zeros(2, *shape, dtype=dtype, device="cuda")[1]
        t.untyped_storage().resize_(0)
        return t
    q, kv = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: RotaryEmbedding(64)(freed(2, 1, 2, 64)), lambda: cache.attention(freed(2, 1, 2, 64), table, lens),
                 lambda: cache.attention(q, table, lens, out=freed(2, 1, 2, 64)), lambda: cache.append(freed(2, 1, 2, 64), kv, table, lens),
                 lambda: cache.append(kv, freed(2, 1, 2, 64), table, lens)):
        with pytest.raises(ValueError, match="no memory"):
            call()
    for args in ((freed(2, 2, dtype=torch.int32), lens, None), (table, freed(2, dtype=torch.int32), None), (table, lens, freed(3, dtype=torch.int32))):
        with pytest.raises((ValueError, RuntimeError)):
            cache.attention(q[:, 0] if args[2] is not None else q, *args)
    leaf = torch.ones(2, 3, 2, 64, device="cuda", requires_grad=True)
    y = RotaryEmbedding(64)(leaf)
    (d,) = torch.autograd.grad(y, leaf, torch._efficientzerotensor(2, 3, 2, 64, device="cuda"))
    assert bool((d == 0).all())


def overwrite_what_is_free():
    """Blocks of the size of a small table, from the current stream's memory, with other contents."""
    return [torch.full((n,), -(2 ** 61) + 12345, dtype=torch.int64, device="cuda") for n in (32, 64) for _ in range(200)]


def test_frequencies_outlive_their_embedding_on_other_streams():
    """First call on one stream, another behind a long kernel on a second one, the embedding gone, new memory on the first."""
    x = draw((40, 4, 64), torch.bfloat16, 3).cuda()
    want = RotaryEmbedding(64, base=777.0)(x)
    gc.collect()
    torch.cuda.synchronize()
    rope, side = RotaryEmbedding(64, base=777.0), torch.cuda.Stream()
    rope(x)
    cache = PagedKVCache.allocate(4, 16, 4, 64)
    table, lens = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), torch.tensor([40], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)   # a tenth of a second
        got = rope(x)
        cache.append(x.unsqueeze(0), x.unsqueeze(0), table, lens, rotary=rope)
    del rope
    gc.collect()
    other = overwrite_what_is_free()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(cache.read(table, lens, 40)[0][0], want) and len(other) == 400


def test_frequencies_outlive_their_embedding_in_a_graph():
    x = draw((40, 4, 64), torch.bfloat16, 4).cuda()
    rope, g = RotaryEmbedding(64, base=555.0), torch.cuda.CUDAGraph()
    want = rope(x)
    with torch.cuda.graph(g):
        got = rope(x)
    del rope
    gc.collect()
    other = overwrite_what_is_free()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(other) == 400


# ---------------------------------------------------------------------------------------------------------------
# attention over a cache
# ---------------------------------------------------------------------------------------------------------------

def filled(lens, Hkv, D, page, dtype, codes, seed):
    """(cache, block_table, cache_seqlens) of random tokens, the pages in random order."""
    g = torch.Generator().manual_seed(seed)
    blocks = -(-max(max(lens), 1) // page)
    cache = PagedKVCache.allocate(len(lens) * blocks, page, Hkv, D, torch.float8_e4m3fn if codes else dtype)
    table = torch.randperm(len(lens) * blocks, generator=g).view(len(lens), blocks).int().cuda()
    seqlens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(len(lens), max(lens), Hkv, D, generator=g).to(dtype).cuda() for _ in range(2))
    full = torch.full_like(seqlens, max(lens))
    cache.append(k, v, table, full)
    return cache, table, seqlens


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("H,lens,rows,backwards,forwards", [(4, [3000, 2000, 2500], 25, [0, 10, 5, 20], [0, 10, 10, 20]), (40, [1500, 700, 1900], 25, [0, 10, 5, 20], [0, 10, 10, 20]),
                                                            (4, [3000, 2000, 2500], 5, [0, 3, 1, 4], [0, 3, 3, 4]), (4, [300, 200, 250], 5, [0, 3, 1, 4], [0, 3, 3, 4])])
def test_first_rows_that_go_backwards(codes, H, lens, rows, backwards, forwards):
    """They count as their predecessors, in units that several blocks share as in whole ones: no row is two sequences'."""
    cache, table, seqlens = filled(lens, 1, 64, 16, torch.bfloat16, codes, 61)
    q, n = draw((rows, H, 64), torch.bfloat16, 62).cuda(), forwards[-1]
    results = []
    for first in (backwards, forwards):
        out = torch.full_like(q, 7.0)
        cu = torch.tensor(first, dtype=torch.int32, device="cuda")
        o, lse = cache.attention(q, table, seqlens, cu_seqlens=cu, out=out, return_lse=True)
        assert lib.last_device_status() == 0
        results.append((o, lse[:, :n]))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    assert bool((results[0][0][n:] == 7.0).all()) and bool((results[0][0][:n] != 7.0).any(2).all())


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("n", [1, 3, 70])
@pytest.mark.parametrize("axis", [0, 1, 2])
def test_queries_in_memory_that_several_share(codes, n, axis):
    """q expanded over sequences, positions or heads: as its copy, whichever kernel it takes; packed too."""
    cache, table, seqlens = filled([300, 90, 1000], 2, 64, 16, torch.float16, codes, 63)
    shape = [3, n, 4, 64]
    q = draw([1 if i == axis else x for i, x in enumerate(shape)], torch.float16, 64).cuda().expand(shape)
    got, want = (cache.attention(t, table, seqlens, return_lse=True) for t in (q, q.clone(memory_format=torch.contiguous_format)))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if axis > 0:
        cu = torch.tensor([0, 0, n, n], dtype=torch.int32, device="cuda")
        packed = q[1]
        got, want = (cache.attention(t, table, seqlens, cu_seqlens=cu, return_lse=True) for t in (packed, packed.clone(memory_format=torch.contiguous_format)))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert lib.last_device_status() == 0


def test_sizes_beyond_the_kernels_are_refused_by_name():
    """Before anything is launched or allocated: the operands are one row in the place of many."""
    cache = PagedKVCache.allocate(1, 1 << 20, 1, 64, torch.float8_e4m3fn)
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    for blocks, seq, word in ((1024, 1, "2\\^30 - 1 tokens"), (1, 1 << 30, "2\\^30 - 1 new tokens"), (512, 1 << 20, "too long")):
        table = torch.zeros(1, blocks, dtype=torch.int32, device="cuda")
        with pytest.raises(ValueError, match=word):
            cache.attention(q.expand(1, seq, 1, 64), table, lens)
    for bad in (q[..., :0], q[..., :32], q[0, 0, 0, 0]):
        with pytest.raises(ValueError):
            cache.attention(bad, table, lens)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("n", [3, 70])
def test_rows_at_negative_positions(codes, n):
    """More new tokens than tokens: causal rows in front of the sequence see nothing, others see every key."""
    cache, table, seqlens = filled([2, 0, 300], 1, 64, 16, torch.bfloat16, codes, 65)
    q = draw((3, 1, 2, 64), torch.bfloat16, 66).expand(3, n, 2, 64).contiguous().cuda()
    o, lse = cache.attention(q, table, seqlens, return_lse=True)
    assert bool((o[0, :n - 2] == 0).all()) and bool((lse[0, :, :n - 2] == -torch.inf).all()) and bool(lse[0, :, n - 2:].isfinite().all())
    o, lse = cache.attention(q, table, seqlens, causal=False, return_lse=True)
    for b in (0, 2):   # the same query everywhere: the same row everywhere
        assert torch.equal(o[b], o[b, -1:].expand_as(o[b])) and bool(lse[b].isfinite().all())
    assert bool((o[1] == 0).all()) and bool((lse[1] == -torch.inf).all())


# ---------------------------------------------------------------------------------------------------------------
# what a cache holds
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("codes", [False, True])
def test_a_cache_holds_the_turned_keys_and_the_values(codes):
    """Step by step as a server appends, against the rows that were given, turned by their positions in 64 bits.  16 bits: keys as in
    test_rotary_gpu.py, values equal.  8 bits: half a step of the code (2^-4 of the value, or 2^-16 of the row's largest where codes are
    subnormal: half of 2^-9 steps of 2^e, 2^e < largest / 224), plus for keys what the angle may be off, twice where the code flips."""
    Hkv, D, page, dtype = 2, 64, 16, torch.bfloat16
    cache = PagedKVCache.allocate(20, page, Hkv, D, torch.float8_e4m3fn if codes else dtype)
    rope = RotaryEmbedding(D, base=5000.0)
    table = torch.randperm(20, generator=torch.Generator().manual_seed(71))[:14].view(2, 7).int().cuda()
    rows = {(w, b): [] for w in "kv" for b in (0, 1)}
    total = [0, 0]
    for step, news in enumerate(([60, 17], [23, 41], [1, 1], [0, 1], [1, 0])):
        total = [a + b for a, b in zip(total, news)]
        lens, cu = torch.tensor(total, dtype=torch.int32).cuda(), torch.tensor([0, news[0], sum(news)], dtype=torch.int32).cuda()
        k, v = (draw((sum(news), Hkv, D), dtype, 72 + 2 * step + i) for i in (0, 1))
        cache.append(k.cuda(), v.cuda(), table, lens, cu_seqlens=cu, rotary=rope)
        for w, x in (("k", k), ("v", v)):
            for b, part in enumerate(x.split(news)):
                rows[w, b].append(part)
        kk, vv = (t.cpu().double() for t in cache.read(table, lens, max(total)))
        for b in (0, 1):
            given = torch.cat(rows["k", b])
            want = pm.rotary(given, torch.arange(total[b]), rope.frequencies)
            pair = (given[..., :D // 2].double().abs() + given[..., D // 2:].double().abs()).repeat(1, 1, 2) * 2.0 ** -20
            values = torch.cat(rows["v", b]).double()
            if codes:
                def half(x):
                    return torch.maximum(x.abs() * 2.0 ** -4, x.abs().amax(-1, keepdim=True) * 2.0 ** -16)
                assert bool(((kk[b, :total[b]] - want).abs() <= half(want) + 2 * pair).all())
                assert bool(((vv[b, :total[b]] - values).abs() <= half(values)).all())
            else:
                assert bool(((kk[b, :total[b]] - want).abs() <= want.abs() * 2.0 ** -8 + pair).all())
                assert torch.equal(vv[b, :total[b]], values)
            if total[b] > 1:   # a tolerance that tells: the rows as they were given are outside of it
                assert bool(((kk[b, :total[b]] - given.double()).abs() > 0.5).any())
    assert lib.last_device_status() == 0


def test_codes_that_are_written_again_stay():
    """Reading codes back and writing them gives the same codes and scales; a row whose largest code is 224 may take the next smaller
    scale (448 of it is the same value), with codes of twice the value."""
    cache, table, lens = filled([77, 77], 2, 128, 16, torch.bfloat16, True, 74)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    a, b = cache.read(table, lens, 77)
    cache.append(a, b, table, lens)
    for i, values in ((0, a), (1, b)):
        pool, scale = (cache.k, cache.k_scale) if i == 0 else (cache.v, cache.v_scale)
        borderline = before[i].float().abs().amax(-1) == 224
        assert int(borderline.sum()) < borderline.numel() // 4
        assert torch.equal(pool.view(torch.uint8)[~borderline], before[i].view(torch.uint8)[~borderline])
        assert torch.equal(scale.view(torch.uint8)[~borderline], before[2 + i].view(torch.uint8)[~borderline])
        assert torch.equal(cache.read(table, lens, 77)[i], values)
    assert lib.last_device_status() == 0
