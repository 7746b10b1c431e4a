"""Writing into paged caches, reading them back and attention over them on the GPU, against the 64-bit oracle.

Tolerances.  Written rows: one rounding of a 16-bit type, and for turned keys 2^-20 of the pair's magnitudes (test_rotary_gpu.py);
8-bit rows that are not turned are equal to the oracle's, codes and scales.  Rows read back are equal (a code times a power of two
is exact).  Attention: u = half a step of the type; each probability is rounded by u (fp16: or by 2^-25 of the largest, n of them), the result by u,
and 32-bit scores, exponentials and sums add 2^-16 of the magnitudes A = sum p |v|: |o - o*| <= u (A + |o*|) + 2^-16 A + n 2^-25 max |v|.
lse: 2^-17 (1 + |lse|)."""

import ctypes
import math
import random

import pytest
import torch

from attn_engine import PagedKVCache, RotaryEmbedding
from core.native import lib
from examples_b200 import programs
from oracle import paged_math as pm

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator().manual_seed(seed)


class Case:
    """A cache on the CPU and on the GPU whose rows behind the sequences' ends are NaN, and whose table is garbage there."""

    def __init__(self, lens, Hkv, D, page, dtype=torch.bfloat16, codes=False, seed=0, hnd=True, more_blocks=2, spare=2):
        g = gen(seed)
        self.lens, self.page, self.Hkv, self.D, self.dtype, self.codes = lens, page, Hkv, D, dtype, codes
        need = [-(-n // page) for n in lens]
        blocks = max(max(need), 1) + more_blocks
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).tolist()
        self.table = torch.full((len(lens), blocks), -1, dtype=torch.int32)
        self.table[:, max(need):] = 1 << 30
        x = [torch.randn(pages, page, Hkv, D, generator=g).to(dtype) for _ in range(2)]
        used = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(need):
            for i in range(n):
                p = order.pop()
                self.table[b, i] = p
                used[p, :min(page, lens[b] - i * page)] = True
        self.used = used
        if codes:
            self.pools, self.scales = [], []
            for t in x:
                c = (t.float() * 100).clamp(-448, 448).to(E4M3)
                s = torch.randint(117, 122, (pages, page, Hkv), generator=g, dtype=torch.uint8)
                c.view(torch.uint8)[~used] = 0x7f
                s[~used] = 255
                self.pools.append(c)
                self.scales.append(s)
        else:
            self.scales = [None, None]
            for t in x:
                t[~used] = float("nan")
            self.pools = x

        def dev(t):
            if t is None:
                return None
            t = t.cuda()
            return t.transpose(1, 2).contiguous().transpose(1, 2) if hnd else t
        self.cache = PagedKVCache(dev(self.pools[0]), dev(self.pools[1]), dev(self.scales[0]), dev(self.scales[1]))
        self.cache_seqlens = torch.tensor(lens, dtype=torch.int32).cuda()
        self.block_table = self.table.cuda()

    def sequence(self, which, b):
        return pm.sequence(self.pools[which], self.scales[which], self.table[b], self.lens[b])


def fresh_rows(news, shape, dtype, packed, seed, pad=0):
    """(rows on the CPU [sum(news) (+ pad), ...], as the call takes them, cu_seqlens or None)"""
    rows = torch.randn(sum(news) + pad, *shape, generator=gen(seed)).to(dtype)
    if packed:
        cu = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32)
        return rows, rows.cuda(), cu.cuda()
    return rows, rows.view(len(news), news[0], *shape).cuda(), None


# ---------------------------------------------------------------------------------------------------------------
# writing
# ---------------------------------------------------------------------------------------------------------------

def check_append(c, news, k, v, rope=None):
    assert lib.last_device_status() == 0
    page, first = c.page, 0
    want = [p.clone() for p in c.pools]
    bytes_ = [None if s is None else s.clone() for s in c.scales]
    turned = torch.zeros(c.pools[0].shape[:2], dtype=torch.bool)
    exact, pair = torch.zeros(c.pools[0].shape, dtype=torch.float64), torch.zeros(c.pools[0].shape, dtype=torch.float64)
    for b, n in enumerate(news):
        for i in range(n):
            t = c.lens[b] - n + i
            if t < 0 or t // page >= c.table.shape[1]:
                continue
            p = int(c.table[b, t // page])
            if not 0 <= p < want[0].shape[0]:
                continue
            for w, rows in enumerate((k, v)):
                x = rows[first + i]
                if w == 0 and rope is not None:
                    turned[p, t % page] = True
                    exact[p, t % page] = pm.rotary(x, torch.tensor(t), rope.frequencies, rope.magnitude, rope.interleaved)
                    pair[p, t % page] = x.double().abs().amax(-1, keepdim=True) * 2 * rope.magnitude
                elif not c.codes:
                    want[w][p, t % page] = x
                else:
                    for h in range(c.Hkv):
                        codes, byte = pm.quantise(x[h])
                        want[w][p, t % page, h] = codes
                        bytes_[w][p, t % page, h] = byte
        first += n

    def bits(t):
        return t.contiguous().view(torch.uint8 if t.element_size() == 1 else torch.int16)
    got = [c.cache.k.cpu(), c.cache.v.cpu()]
    got_s = [None if s is None else s.cpu().view(torch.uint8) for s in (c.cache.k_scale, c.cache.v_scale)]
    assert torch.equal(bits(got[1]), bits(want[1]))
    assert torch.equal(bits(got[0])[~turned], bits(want[0])[~turned])
    if c.codes:
        assert torch.equal(got_s[1], bytes_[1]) and torch.equal(got_s[0][~turned], bytes_[0][~turned])
    if rope is not None and bool(turned.any()):
        e, m = exact[turned], pair[turned] * 2.0 ** -20
        if c.codes:
            e8 = got_s[0][turned].double() - 127
            for top, byte in zip(e.abs().amax(-1).flatten().tolist(), got_s[0][turned].flatten().tolist()):
                assert byte - 127 in (pm.exponent_of(top * (1 - 2.0 ** -19)), pm.exponent_of(top * (1 + 2.0 ** -19)))
            step = torch.exp2(e8).unsqueeze(-1)
            val = got[0][turned].float().double() * step
            tol = torch.maximum(e.abs() * 2.0 ** -4, step * 2.0 ** -10) + 2 * m
        else:
            val, tol = got[0][turned].double(), e.abs() * (torch.finfo(c.dtype).eps / 2) + m + (2.0 ** -24 if c.dtype == torch.float16 else 0.0)
        assert bool(((val - e).abs() <= tol).all())


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("dtype,D,page,hnd", [(torch.bfloat16, 128, 64, True), (torch.float16, 64, 16, False), (torch.bfloat16, 64, 8, True), (torch.float16, 128, 256, True)])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("rotary", [None, "half", "interleaved", "part"])
def test_append(codes, dtype, D, page, hnd, packed, rotary):
    news = [5, 1, 70, 0, 3] if packed else [4, 4, 4]
    lens = [5, 300, 131, 40, 3][:len(news)] if packed else [4, 260, 33]
    c = Case(lens, 3, D, page, dtype, codes, seed=31, hnd=hnd)
    rope = {None: None, "half": RotaryEmbedding(D), "interleaved": RotaryEmbedding(D, interleaved=True),
            "part": RotaryEmbedding(D // 4 if D == 128 else 16, scaling="yarn", factor=8.0)}[rotary]
    k, kd, cu = fresh_rows(news, (3, D), dtype, packed, 32, pad=3 if packed else 0)
    v, vd, _ = fresh_rows(news, (3, D), dtype, packed, 33, pad=3 if packed else 0)
    c.cache.append(kd, vd, c.block_table, c.cache_seqlens, cu_seqlens=cu, rotary=rope)
    check_append(c, news, k, v, rope)


def test_append_rows_of_extreme_values():
    """Zeros, one value, the largest and smallest, subnormals, infinities and NaN; each row by itself."""
    D = 64
    c = Case([16], 1, D, 16, torch.bfloat16, True, seed=34)
    k = torch.zeros(16, 1, D)
    k[1, 0, 3] = 448.0
    k[2, 0, 5] = -450.0
    k[3] = 3.3e38
    k[4] = 1e-38 * torch.randn(D, generator=gen(1))
    k[5] = 1e-40
    k[6, 0, 0] = float("inf")
    k[7, 0, 9] = float("nan")
    k[8, 0, 9] = -float("inf")
    k[9] = torch.randn(D, generator=gen(2)) * 1e5
    k[10] = 1.75
    k[11] = 1.7578125
    k[12] = torch.arange(D) * 7.0     # ties of the codes
    k[13] = torch.linspace(-464, 464, D)
    k[14, 0, 1] = -0.0
    k[15] = 2.0 ** -126
    k = k.to(torch.bfloat16)
    c.cache.append(k.unsqueeze(0).cuda(), k.flip(0).unsqueeze(0).cuda(), c.block_table, c.cache_seqlens)
    check_append(c, [16], k, k.flip(0))


def test_append_of_strided_rows_and_tokens_without_a_place():
    """k and v as slices of one projection; a sequence shorter than its new tokens; a length past the table; pages that do not exist."""
    B, T, Hkv, D, page = 4, 6, 2, 64, 8
    c = Case([3, 50, 20, 0], Hkv, D, page, torch.float16, False, seed=35)
    c.lens = [3, 50, 20, 0]
    c.table[1, 50 // page] = -7          # the last page of sequence 1 does not exist
    c.table[2, 2] = c.pools[0].shape[0]   # one past the last
    wide = torch.randn(B, T, 3 * Hkv, D, generator=gen(36)).half()
    k, v = wide[:, :, Hkv:2 * Hkv], wide[:, :, 2 * Hkv:]
    dev = wide.cuda()
    c.cache.append(dev[:, :, Hkv:2 * Hkv], dev[:, :, 2 * Hkv:], c.table.cuda(), c.cache_seqlens)
    check_append(c, [T] * B, k.flatten(0, 1), v.flatten(0, 1))
    # a length past the table
    c2 = Case([30], 1, D, 16, torch.float16, False, seed=37, more_blocks=0)
    c2.lens = [40]
    k = torch.randn(20, 1, D, generator=gen(38)).half()
    c2.cache.append(k.unsqueeze(0).cuda(), k.unsqueeze(0).cuda(), c2.block_table, torch.tensor([40], dtype=torch.int32).cuda())
    check_append(c2, [20], k, k)


# ---------------------------------------------------------------------------------------------------------------
# reading back
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("dtype,D,page", [(torch.bfloat16, 128, 16), (torch.float16, 64, 128), (torch.float16, 128, 8)])
@pytest.mark.parametrize("max_len", [1, 50, 260])
def test_read(codes, dtype, D, page, max_len):
    c = Case([0, 1, 255, 50, 17], 2, D, page, dtype, codes, seed=41)
    k, v = c.cache.read(c.block_table, c.cache_seqlens, max_len, dtype=dtype)
    assert lib.last_device_status() == 0 and k.dtype == dtype and k.shape == (5, max_len, 2, D)
    for w, got in enumerate((k, v)):
        for b, n in enumerate(c.lens):
            m = min(n, max_len)
            assert torch.equal(got[b, :m].cpu(), c.sequence(w, b)[:m].to(dtype))
            assert bool((got[b, m:] == 0).all())


def test_read_nan_rows_large_scales_and_missing_pages():
    c = Case([40], 1, 64, 8, torch.bfloat16, True, seed=42)
    p = [int(x) for x in c.table[0, :5]]
    c.scales[0][p[0], 0, 0], c.scales[0][p[0], 1, 0], c.scales[0][p[0], 2, 0], c.scales[0][p[0], 3, 0] = 255, 0, 1, 246
    c.cache.k_scale.copy_(c.scales[0].cuda())
    c.table[0, 1], c.table[0, 2] = -1, c.pools[0].shape[0]
    k, _ = c.cache.read(c.table.cuda(), c.cache_seqlens, 40)
    want = c.sequence(0, 0)
    got = k[0].cpu()
    assert bool(got[0].isnan().all()) and torch.equal(got[1:], want[1:].to(torch.bfloat16)) and bool((got[8:24] == 0).all())


def test_what_is_written_is_read():
    """Quantised values are what reading gives back, to the bit, and quantising them again changes nothing."""
    c = Case([77, 12], 2, 128, 16, torch.bfloat16, True, seed=43)
    news = [77, 12]
    k, kd, cu = fresh_rows(news, (2, 128), torch.bfloat16, True, 44)
    c.cache.append(kd, kd, c.block_table, c.cache_seqlens, cu_seqlens=cu)
    a, b = c.cache.read(c.block_table, c.cache_seqlens, 77)
    assert torch.equal(a, b)
    packed = torch.cat([a[0], a[1, :12]])
    err = (packed.cpu().double() - k.double()).abs()
    assert bool((err <= torch.maximum(k.double().abs() * 2.0 ** -4, k.double().abs().amax(-1, keepdim=True) * 2.0 ** -17)).all())
    before = c.cache.k.clone()
    c.cache.append(packed, packed, c.block_table, c.cache_seqlens, cu_seqlens=cu)
    again, _ = c.cache.read(c.block_table, c.cache_seqlens, 77)
    assert torch.equal(again, a) and before.shape == c.cache.k.shape


# ---------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------

def check_attention(c, news, q, o, lse, packed, H, causal=True, window=None, scale=None):
    assert lib.last_device_status() == 0
    u = torch.finfo(c.dtype).eps / 2
    scale = c.D ** -0.5 if scale is None else scale
    o, lse = o.cpu().double().reshape(-1, H, c.D), lse.cpu().double()
    first = 0
    for b, n in enumerate(news):
        if n == 0:
            continue
        k, v = c.sequence(0, b), c.sequence(1, b)
        want, want_lse, mag = pm.attention(q[first:first + n], k, v, c.lens[b], n, scale, causal, window)
        got, got_lse = o[first:first + n], lse[:, first:first + n] if packed else lse[b]
        top = float(v.abs().max()) if c.lens[b] else 0.0
        tol = u * (mag + want.abs()) + 2.0 ** -16 * mag + c.lens[b] * 2.0 ** -25 * top + (2.0 ** -25 if c.dtype == torch.float16 else 0.0)
        assert bool(((got - want).abs() <= tol).all()), (b, ((got - want).abs() - tol).max().item())
        none = want_lse == -math.inf
        assert torch.equal(none, got_lse == -math.inf)
        assert bool(((got_lse - want_lse).abs() <= 2.0 ** -17 * (1 + want_lse.abs()))[~none].all()), b
        assert bool((got[none.T] == 0).all())
        first += n


def run_attention(lens, news, H, Hkv, D, page, dtype=torch.bfloat16, codes=False, packed=False, seed=0, hnd=True, pad=0, **kwargs):
    c = Case(lens, Hkv, D, page, dtype, codes, seed=seed + 51, hnd=hnd)
    q, qd, cu = fresh_rows(news, (H, D), dtype, packed, seed + 52, pad)
    o, lse = c.cache.attention(qd, c.block_table, c.cache_seqlens, cu_seqlens=cu, return_lse=True, **kwargs)
    check_attention(c, news, q, o, lse, packed, H, **{k: v for k, v in kwargs.items() if k in ("causal", "window", "scale")})
    return c, q, o, lse


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("dtype,D,page", [(torch.bfloat16, 128, 64), (torch.float16, 64, 16), (torch.float16, 128, 8), (torch.bfloat16, 64, 256), (torch.bfloat16, 128, 128)])
@pytest.mark.parametrize("H,Hkv", [(4, 1), (6, 2), (2, 2)])
def test_single_tokens(codes, dtype, D, page, H, Hkv):
    run_attention([1, 7, 128, 129, 300, 1000], [1] * 6, H, Hkv, D, page, dtype, codes)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("dtype,D,page", [(torch.bfloat16, 128, 32), (torch.float16, 64, 64)])
@pytest.mark.parametrize("causal,window", [(True, None), (False, None), (True, 1), (True, 50), (True, 200)])
def test_chunks(codes, dtype, D, page, causal, window):
    run_attention([37, 150, 290], [37] * 3, 4, 2, D, page, dtype, codes, causal=causal, window=window)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("window", [None, 33])
def test_packed_mixture_leaves_padding_alone(codes, window):
    """Chunks, single tokens, sequences without new ones; rows behind the last are left as they were."""
    lens, news = [200, 1, 333, 64, 500, 130], [150, 1, 0, 3, 1, 130]
    H, D = 6, 64
    c = Case(lens, 2, D, 16, torch.float16, codes, seed=61)
    q, qd, cu = fresh_rows(news, (H, D), torch.float16, True, 62, pad=9)
    out = torch.full_like(qd, 7.0)
    got, lse = c.cache.attention(qd, c.block_table, c.cache_seqlens, cu_seqlens=cu, window=window, out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr() and bool((out[sum(news):] == 7.0).all())
    check_attention(c, news, q, got, lse, True, H, window=window)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("D,window", [(64, None), (64, 700), (128, None)])
def test_long_packed_mixtures(codes, D, window):
    """Single tokens on long contexts in units of many rows, most of which are nobody's: warps without a row keep in step with the
    others of their tile.  Several calls, which agree to the bit."""
    news = [40, 1, 1, 5, 1, 33, 1, 1]
    lens = [1500, 1900, 700, 1200, 2300, 900, 1601, 130]
    c, q, o, lse = run_attention(lens, news, 8, 2, D, 16, torch.float16, codes, packed=True, seed=9, window=window)
    cu = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32).cuda()
    for _ in range(20):
        again, lse2 = c.cache.attention(q.cuda(), c.block_table, c.cache_seqlens, cu_seqlens=cu, window=window, return_lse=True)
        assert torch.equal(again, o) and torch.equal(lse2, lse)
    assert lib.last_device_status() == 0


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("group", [1, 3, 5, 7, 16, 33, 64, 128])
def test_group_sizes(codes, group):
    run_attention([40, 150], [9, 9], group, 1, 64, 16, torch.bfloat16, codes, seed=group)


@pytest.mark.parametrize("codes", [False, True])
def test_rows_that_see_nothing(codes):
    """Empty sequences, and more new tokens than tokens: 0 and -inf."""
    c, q, o, lse = run_attention([0, 5, 2, 300], [4] * 4, 4, 2, 128, 16, torch.bfloat16, codes)
    assert bool((o[0] == 0).all()) and bool((lse[0] == -math.inf).all()) and bool((o[2, :2] == 0).all())
    run_attention([0, 5, 2, 300], [4] * 4, 4, 2, 64, 16, torch.float16, codes, causal=False)


@pytest.mark.parametrize("codes", [False, True])
def test_long_contexts_are_split_and_merged(codes):
    """One sequence over all SMs, with a window that begins inside a share, and chunks whose units are cut."""
    run_attention([5000], [1], 4, 1, 128, 64, torch.bfloat16, codes, seed=3)
    run_attention([5000], [3], 2, 1, 64, 16, torch.float16, codes, seed=4, window=3001)
    run_attention([2000, 900], [64, 64], 4, 2, 64, 64, torch.bfloat16, codes, seed=5)


@pytest.mark.parametrize("codes", [False, True])
def test_large_scores_and_growing_maxima(codes):
    """Scores that grow along the sequence move the running maximum again and again; a scale of its own."""
    c = Case([700], 1, 64, 16, torch.float16, codes, seed=71)
    t = torch.arange(700)
    order = c.table[0].long()
    for w in range(1):
        grow = (t / 100.0).view(-1, 1, 1)
        base = torch.ones(700, 1, 64) * grow
        if codes:
            c.pools[0][order[t // 16], t % 16] = base.to(E4M3)
            c.scales[0][order[t // 16], t % 16] = 127
            c.cache.k_scale.copy_(c.scales[0].cuda())
        else:
            c.pools[0][order[t // 16], t % 16] = base.half()
    c.cache.k.copy_(c.pools[0].cuda())
    q = torch.cat([torch.full((1, 2, 64), 1.0), torch.full((1, 2, 64), -1.0), torch.randn(3, 2, 64, generator=gen(72))]).half()
    o, lse = c.cache.attention(q.unsqueeze(0).cuda(), c.block_table, c.cache_seqlens, scale=0.5, return_lse=True)
    check_attention(c, [5], q, o, lse, False, 2, scale=0.5)


def test_pools_of_any_strides():
    """K and V as halves of one tensor, heads in front of rows or behind them, a table that is a slice of a wider one, heads-first q."""
    for hnd in (False, True):
        run_attention([130, 77], [3, 3], 4, 2, 64, 32, hnd=hnd)
    c = Case([130, 77], 2, 64, 32, torch.bfloat16, False, seed=81)
    both = torch.stack([c.cache.k, c.cache.v], 1)   # [pages, 2, page, heads, D]
    cache = PagedKVCache(both[:, 0], both[:, 1])
    wide = torch.full((2, 40), 5, dtype=torch.int32)
    wide[:, 3:3 + c.table.shape[1]] = c.table
    q, _, _ = fresh_rows([3, 3], (4, 64), torch.bfloat16, False, 82)
    qd = q.view(2, 3, 4, 64).transpose(1, 2).contiguous().cuda().transpose(1, 2)
    o, lse = cache.attention(qd, wide.cuda()[:, 3:3 + c.table.shape[1]], c.cache_seqlens, return_lse=True)
    check_attention(c, [3, 3], q, o, lse, False, 4)
    out = torch.zeros(2, 4, 3, 80, dtype=torch.bfloat16, device="cuda").transpose(1, 2)[..., 8:72]
    o2 = cache.attention(qd, wide.cuda()[:, 3:3 + c.table.shape[1]], c.cache_seqlens, out=out)
    assert torch.equal(o2, o)


def test_shared_pages_and_missing_pages():
    """Two sequences with one prefix; pages that do not exist read as zeros."""
    c = Case([64, 64], 1, 64, 16, torch.bfloat16, False, seed=83)
    c.table[1, :3] = c.table[0, :3]
    c.table[0, 1], c.table[1, 2] = -1, 1 << 29
    q, qd, _ = fresh_rows([2, 2], (2, 64), torch.bfloat16, False, 84)
    o, lse = c.cache.attention(qd, c.table.cuda(), c.cache_seqlens, return_lse=True)
    check_attention(c, [2, 2], q, o, lse, False, 2)


def test_freed_pages_in_front_of_a_window():
    """A server frees pages that no window reaches: their entries, and the rows in front of the window, may hold anything."""
    for codes in (False, True):
        c = Case([400], 1, 64, 16, torch.float16, codes, seed=85)
        q, qd, _ = fresh_rows([2], (2, 64), torch.float16, False, 86)
        o, lse = c.cache.attention(qd, c.block_table, c.cache_seqlens, window=40, return_lse=True)
        check_attention(c, [2], q, o, lse, False, 2, window=40)
        bad = c.table.clone()
        bad[0, :(400 - 2 + 1 - 40) // 16] = -1
        again, lse2 = c.cache.attention(qd, bad.cuda(), c.cache_seqlens, window=40, return_lse=True)
        assert torch.equal(again, o) and torch.equal(lse2, lse)
        if not codes:
            first = 400 - 2 + 1 - 40   # the first key of the first row
            k, v = c.cache.k.clone(), c.cache.v.clone()
            for t in range(first):
                p = int(c.table[0, t // 16])
                k[p, t % 16] = float("nan")
                v[p, t % 16] = float("inf")
            again = PagedKVCache(k, v).attention(qd, c.block_table, c.cache_seqlens, window=40)
            assert torch.equal(again, o)


def test_codes_of_extreme_rows():
    """Factors outside the 16-bit format's own range, a NaN row, zeros."""
    for dtype in (torch.bfloat16, torch.float16):
        c = Case([50], 1, 64, 16, dtype, True, seed=87)
        p, r = int(c.table[0, 0]), 3
        c.scales[1][p, r, 0] = 150 if dtype == torch.bfloat16 else 133    # values up to 448 * 2^23, 2^6
        c.scales[1][p, r + 1, 0] = 0 if dtype == torch.bfloat16 else 110
        c.pools[1].view(torch.uint8)[p, r + 2, 0] = 0
        c.scales[1][p, r + 2, 0] = 254
        c.cache.v_scale.copy_(c.scales[1].cuda())
        c.cache.v.view(torch.uint8).copy_(c.pools[1].view(torch.uint8).cuda())
        q, qd, _ = fresh_rows([1], (2, 64), dtype, False, 88)
        o, lse = c.cache.attention(qd, c.block_table, c.cache_seqlens, return_lse=True)
        check_attention(c, [1], q, o, lse, False, 2)
        c.cache.v_scale.view(torch.uint8)[p, r, 0] = 255
        assert bool(c.cache.attention(qd, c.block_table, c.cache_seqlens).isnan().all())


def test_results_do_not_change_from_call_to_call():
    c, q, o, lse = run_attention([3000, 700], [5, 5], 4, 1, 128, 64)
    for _ in range(3):
        o2, lse2 = c.cache.attention(q.view(2, 5, 4, 128).cuda(), c.block_table, c.cache_seqlens, return_lse=True)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_many_sequences():
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 40, (1024,), generator=g).tolist()
    run_attention(lens, [1] * 1024, 2, 1, 64, 8, torch.float16)
    c = Case([3] * 1025, 1, 64, 8)
    with pytest.raises(ValueError, match="1024"):
        c.cache.attention(torch.zeros(1025, 1, 1, 64, dtype=torch.bfloat16, device="cuda"), c.block_table, c.cache_seqlens)


# ---------------------------------------------------------------------------------------------------------------
# a step as a server makes it, refusals, streams, graphs
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("codes", [False, True])
def test_steps_of_a_server(codes):
    """Prompts in two chunks, then single tokens, each step rotary -> append -> attention; against attention over everything that
    was appended, as the cache holds it."""
    H, Hkv, D, page, dtype = 4, 2, 64, 16, torch.bfloat16
    cache = PagedKVCache.allocate(20, page, Hkv, D, dtype=E4M3 if codes else dtype)
    rope = RotaryEmbedding(D)
    table = torch.randperm(20, generator=gen(91))[:14].view(2, 7).int().cuda()
    total = [0, 0]
    g = torch.Generator(device="cuda").manual_seed(92)
    for news in ([60, 17], [23, 41], [1, 1], [1, 1], [0, 1]):
        total = [a + b for a, b in zip(total, news)]
        rows = sum(news)
        lens, cu = torch.tensor(total, dtype=torch.int32).cuda(), torch.tensor([0, news[0], rows], dtype=torch.int32).cuda()
        pos = torch.cat([torch.arange(t - n, t) for t, n in zip(total, news)]).cuda()
        q, k, v = (torch.randn(rows, h, D, generator=g, device="cuda", dtype=dtype) for h in (H, Hkv, Hkv))
        cache.append(k, v, table, lens, cu_seqlens=cu, rotary=rope)
        o, lse = cache.attention(rope(q, positions=pos), table, lens, cu_seqlens=cu, return_lse=True)
        kk, vv = cache.read(table, lens, max(total))
        qq = rope(q, positions=pos).cpu()
        first = 0
        for b, n in enumerate(news):
            want, want_lse, mag = pm.attention(qq[first:first + n], kk[b, :total[b]].cpu().double(), vv[b, :total[b]].cpu().double(), total[b], n, D ** -0.5)
            got = o[first:first + n].cpu().double()
            assert bool(((got - want).abs() <= 2.0 ** -8 * (mag + want.abs()) + 2.0 ** -16 * mag).all())
            assert bool(((lse[:, first:first + n].cpu().double() - want_lse).abs() <= 2.0 ** -17 * (1 + want_lse.abs())).all())
            first += n
        assert lib.last_device_status() == 0
    if not codes:   # the keys in the cache are the turned ones
        assert total == [85, 61]


def test_refusals():
    c = Case([20, 30], 2, 64, 16)
    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    t, s = c.block_table, c.cache_seqlens
    cu = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    bad_attention = [
        (q, t.long(), s, {}), (q, t, s.long(), {}), (q, t[:1], s, {}), (q, t[0], s, {}), (q, t.cpu(), s, {}), (q, t, s.cpu(), {}), (q[0], t, s, {}),
        (q, t, s, dict(cu_seqlens=cu)), (q[:, 0], t, s, dict(cu_seqlens=cu[:2])), (q[:, 0], t, s, dict(cu_seqlens=cu.long())), (q[:, 0], t, s, {}),
        (q[:1], t, s, {}), (q[:, :, :3], t, s, {}), (q.half(), t, s, {}), (q.float(), t, s, {}), (q[..., :32], t, s, {}), (q.cpu(), t, s, {}),
        (q, t, s, dict(scale=0.0)), (q, t, s, dict(scale=-1.0)), (q, t, s, dict(scale=math.nan)), (q, t, s, dict(scale=math.inf)), (q, t, s, dict(window=0)),
        (q, t, s, dict(window=-3)), (q, t, s, dict(window=5, causal=False)), (q, t, s, dict(out=q[:, :, :2])), (q, t, s, dict(out=q.half())),
        (q.clone().requires_grad_(), t, s, {}), (torch.zeros(2, 1, 4, 66, dtype=torch.bfloat16, device="cuda")[..., 1:65], t, s, {}),
        (torch.zeros(2, 1, 258, 64, dtype=torch.bfloat16, device="cuda"), t, s, {}), (q.transpose(2, 3), t, s, {}), (q, t[:0], s[:0], {})]
    for q_, t_, s_, kw in bad_attention:
        with pytest.raises(ValueError):
            c.cache.attention(q_, t_, s_, **kw)
    bad_append = [(k, k[:, :, :1], {}), (k, k.half(), {}), (k.half(), k.half(), {}), (k[:1], k[:1], {}), (k, k[:, :0], {}), (k.clone().requires_grad_(), k, {}),
                  (k, k, dict(rotary=RotaryEmbedding(24))), (k, k, dict(rotary=RotaryEmbedding(128))), (k[:, 0], k[:, 0], {}), (k, k, dict(cu_seqlens=cu))]
    for k_, v_, kw in bad_append:
        with pytest.raises(ValueError):
            c.cache.append(k_, v_, t, s, **kw)
    for kw in (dict(max_len=-1), dict(max_len=4, dtype=torch.float16), dict(max_len=4, dtype=torch.float32)):
        with pytest.raises(ValueError):
            c.cache.read(t, s, **kw)
    assert lib.last_device_status() == 0


def test_empty_calls():
    c = Case([20, 30], 2, 64, 16)
    before = c.cache.k.clone()
    k = torch.zeros(2, 0, 2, 64, dtype=torch.bfloat16, device="cuda")
    c.cache.append(k, k, c.block_table, c.cache_seqlens)
    o, lse = c.cache.attention(torch.zeros(2, 0, 4, 64, dtype=torch.bfloat16, device="cuda"), c.block_table, c.cache_seqlens, return_lse=True)
    assert o.shape == (2, 0, 4, 64) and lse.shape == (2, 4, 0)
    kk, _ = c.cache.read(c.block_table, c.cache_seqlens, 0)
    assert kk.shape == (2, 0, 2, 64)
    # packed rows that belong to nobody
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.ones(5, 4, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 3.0)
    c.cache.attention(q, c.block_table, c.cache_seqlens, cu_seqlens=cu, out=out)
    c.cache.append(q[:, :2], q[:, :2], c.block_table, c.cache_seqlens, cu_seqlens=cu)
    torch.cuda.synchronize()
    assert bool((out == 3.0).all()) and torch.equal(c.cache.k.nan_to_num(9.0), before.nan_to_num(9.0)) and lib.last_device_status() == 0


@pytest.mark.parametrize("codes", [False, True])
def test_captured_step_follows_the_lengths(codes):
    """One captured step of single tokens, replayed with other lengths, tables and tokens; two graphs over one cache, replayed in turn."""
    H, Hkv, D, page, dtype, B = 4, 2, 64, 16, torch.bfloat16, 3
    made = Case([90, 130, 40], Hkv, D, page, dtype, codes, seed=95)
    rope = RotaryEmbedding(D)
    q, k, v = (torch.zeros(B, 1, h, D, dtype=dtype, device="cuda") for h in (H, Hkv, Hkv))
    lens, table, pos = made.cache_seqlens.clone(), made.block_table.clone(), torch.zeros(B, 1, dtype=torch.int64, device="cuda")

    def step():
        made.cache.append(k, v, table, lens, rotary=rope)
        return made.cache.attention(rope(q, positions=pos), table, lens, return_lse=True)
    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step()))
    gen_ = torch.Generator(device="cuda").manual_seed(96)
    results = []
    for i, n in enumerate(([88, 100, 33], [16, 130, 1], [90, 97, 40])):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen_, device="cuda", dtype=dtype))
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        pos.copy_((lens.long() - 1).unsqueeze(1))
        graphs[i % 2][0].replay()
        torch.cuda.synchronize()
        o, lse = (x.clone() for x in graphs[i % 2][1])
        want = made.cache.attention(rope(q, positions=pos), table, lens, return_lse=True)
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1]) and bool(o.isfinite().all())
        results.append(o)
    assert not torch.equal(results[0], results[1]) and lib.last_device_status() == 0


def test_two_streams_at_once():
    """Calls with workspaces of their own run side by side."""
    made = [run_attention([2000, 50], [3, 3], 4, 2, 64, 16, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for (c, q, _, _), s in zip(made, streams):
            with torch.cuda.stream(s):
                outs.append(c.cache.attention(q.view(2, 3, 4, 64).cuda(), c.block_table, c.cache_seqlens))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, made[i % 2][2])


class _Word:
    """The device status word as an array that torch can write."""

    def __init__(self):
        ptr = ctypes.c_void_p()
        lib.check(lib.load_library().attn_b200_device_status_word(0, ctypes.byref(ptr)), "attn_b200_device_status_word")
        self.__cuda_array_interface__ = {"shape": (1,), "typestr": "<i4", "data": (ptr.value, False), "version": 3}


@pytest.mark.parametrize("codes", [False, True])
def test_calls_behind_a_recorded_failure_leave(codes):
    """The status word says that a wait ran out: the kernels leave; once it has been read the same call is right again."""
    c, q, o, _ = run_attention([500, 2100], [2, 2], 4, 2, 64, 16, codes=codes)
    torch.as_tensor(_Word(), device="cuda").fill_(177)
    c.cache.attention(q.view(2, 2, 4, 64).cuda(), c.block_table, c.cache_seqlens)
    assert lib.last_device_status() == 177
    assert torch.equal(c.cache.attention(q.view(2, 2, 4, 64).cuda(), c.block_table, c.cache_seqlens), o)
    assert lib.last_device_status() == 0


# ---------------------------------------------------------------------------------------------------------------
# layouts and sizes that take the kernels' other paths
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv", [1, 3])
@pytest.mark.parametrize("news", [1, 3, 70])
def test_exponents_that_lie_apart(D, Hkv, news):
    """Scales with the heads behind the rows, which are read byte by byte; one head of rows of a page is one piece otherwise."""
    run_attention([news, 150, 400], [news] * 3, 2 * Hkv, Hkv, D, 16, torch.bfloat16, True, seed=21, hnd=False)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("H,Hkv,news", [(8, 1, 3), (20, 1, 1), (64, 2, 1), (4, 1, 8), (2, 2, 31)])
@pytest.mark.parametrize("lens", [[400, 31, 900], [7000]])
def test_units_of_17_to_32_rows(codes, H, Hkv, news, lens):
    run_attention(lens, [news] * len(lens), H, Hkv, 128, 64, torch.bfloat16, codes, seed=22)
    run_attention(lens, [news] * len(lens), H, Hkv, 64, 16, torch.float16, codes, seed=23, window=205)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_chunks_over_long_contexts(codes, D):
    """Units of two tiles of query rows that are cut between SMs, and one sequence alone."""
    run_attention([4100, 2500], [200, 200], 4, 2, D, 64, torch.bfloat16, codes, seed=24)
    run_attention([6000], [257], 3, 1, D, 16, torch.float16, codes, seed=25, window=4001)
    run_attention([6000], [129], 3, 1, D, 16, torch.float16, codes, seed=26, causal=False)


@pytest.mark.parametrize("codes", [False, True])
def test_many_units_of_one_tile(codes):
    """More units than SMs, none of which is cut: a block takes several, whole."""
    g = gen(27)
    lens = torch.randint(1, 400, (90,), generator=g).tolist()
    run_attention(lens, [1] * 90, 16, 8, 128, 16, torch.bfloat16, codes, seed=27)
    news = [min(n, 1 + i % 50) for i, n in enumerate(lens)]
    run_attention(lens, news, 8, 4, 64, 16, torch.float16, codes, packed=True, seed=28)


@pytest.mark.parametrize("codes", [False, True])
def test_pools_of_more_than_2_to_the_31_values(codes):
    """Pages whose rows lie behind 2^31 values of a pool: written, attended to and read like those of a small one."""
    page, Hkv, D = 256, 8, 128
    pages = 2 ** 31 // (page * Hkv * D) + 9
    lens, news, H = [700, 300], [5, 5], 16
    dtype = torch.float8_e4m3fn if codes else torch.bfloat16
    small = PagedKVCache.allocate(8, page, Hkv, D, dtype)

    def pool(of, *shape):
        big = torch.empty(pages, Hkv, page, *shape, dtype=torch.uint8 if codes else dtype, device="cuda")
        big[-8:] = of.transpose(1, 2).view(big.dtype)
        return big.view(of.dtype).transpose(1, 2)
    sizes = [(small.k, (D,)), (small.v, (D,))] + ([(small.k_scale, ()), (small.v_scale, ())] if codes else [])
    large = PagedKVCache(*[pool(t, *s) for t, s in sizes])
    table = torch.tensor([[6, 1, 7], [3, 0, -1]], dtype=torch.int32, device="cuda")
    seqlens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = []
    for cache, at in ((small, table), (large, torch.where(table >= 0, table + (pages - 8), table))):
        for first, n in ((0, 295), (295, 5)):   # the second sequence's tokens; the first's last 295 and 5
            k, v = (torch.randn(2, n, Hkv, D, generator=gen(31 + first + i)).bfloat16().cuda() for i in range(2))
            cache.append(k, v, at, seqlens if n == 5 else seqlens - 5)
        q = torch.randn(2, 5, H, D, generator=gen(40)).bfloat16().cuda()
        out.append((cache.attention(q, at, seqlens), *cache.read(at, seqlens, 700)))
    assert lib.last_device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(*out)) and bool((out[0][1][0, 405:] != 0).any()) and bool((out[0][0] != 0).any())


# ---------------------------------------------------------------------------------------------------------------
# an engine's program over a cache
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("mask,causal,window", [(None, False, None), (programs.causal, True, None), (programs.sliding_window_mask, True, 128)])
def test_an_engine_reads_a_cache(codes, mask, causal, window):
    eng = programs.masked_softmax_engine(1, 4, 512, 64, 64, mask)
    dtype = eng.dtype
    lens, news = [300, 40, 150], [7, 7, 7]
    c = Case(lens, 2, 64, 16, dtype, codes, seed=91)
    q, qd, _ = fresh_rows(news, (4, 64), dtype, False, 92)
    o = eng.paged_attention(qd, c.cache, c.block_table, c.cache_seqlens)
    (lse,) = eng.last_final_rowscales.values()
    check_attention(c, news, q, o, lse, False, 4, causal=causal, window=window, scale=eng._fparams[0])
    out = torch.empty_like(qd)
    assert eng.paged_attention(qd, c.cache, c.block_table, c.cache_seqlens, out=out) is not None and torch.equal(out, o)


def test_memory_that_a_call_must_not_write_is_refused():
    """Results in memory that several values share, or that a graph holds; pools that want a gradient; q and k turned in one place."""
    c = Case([20, 30], 2, 64, 16)
    q = torch.randn(2, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    t, s = c.block_table, c.cache_seqlens
    for out in (q[:1].expand(2, 1, 4, 64), q.clone().requires_grad_()):
        with pytest.raises(ValueError):
            c.cache.attention(q, t, s, out=out)
    learned = PagedKVCache(c.cache.k.clone().requires_grad_(), c.cache.v.clone())
    for call in (lambda: learned.attention(q, t, s), lambda: learned.read(t, s, 4), lambda: learned.append(kv, kv, t, s)):
        with pytest.raises(ValueError, match="no_grad"):
            call()
    with torch.no_grad():
        assert torch.equal(learned.attention(q, t, s), c.cache.attention(q, t, s))
    with pytest.raises(ValueError, match="same memory"):
        RotaryEmbedding(64)(q, q, inplace=True)
    own = q.clone()
    assert torch.equal(c.cache.attention(own, t, s, out=own), c.cache.attention(q, t, s))   # in q's place


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [1, 40, 3, 7]])
def test_padding_rows_may_hold_anything(codes, news):
    """Rows of q behind the last sequence that are NaN or infinite touch no row of a sequence, in the tile they share with its last ones."""
    lens, H, D, pad = [30, 300, 129, 64], 8, 64, 5
    c = Case(lens, 2, D, 16, torch.float16, codes, seed=93)
    q, qd, cu = fresh_rows(news, (H, D), torch.float16, True, 94, pad)
    qd[sum(news):sum(news) + 3] = float("nan")
    qd[sum(news) + 3:] = float("inf")
    o, lse = c.cache.attention(qd, c.block_table, c.cache_seqlens, cu_seqlens=cu, return_lse=True)
    check_attention(c, news, q[:sum(news)], o[:sum(news)], lse, True, H)


def test_windows_of_any_size():
    """A window as long as numbers go is none, chunks and single tokens, more new tokens than tokens among them."""
    for news in ([9, 9], [1, 1]):
        c = Case([5, 300], 1, 64, 16, torch.bfloat16, False, seed=95)
        q, qd, _ = fresh_rows(news, (4, 64), torch.bfloat16, False, 96)
        plain = c.cache.attention(qd, c.block_table, c.cache_seqlens, return_lse=True)
        for window in (301, 1 << 29, 2 ** 31 - 1, 2 ** 40):
            wide = c.cache.attention(qd, c.block_table, c.cache_seqlens, window=window, return_lse=True)
            check_attention(c, news, q, *wide, False, 4)
            assert torch.equal(wide[1] == -math.inf, plain[1] == -math.inf)


@pytest.mark.parametrize("seed", range(40))
def test_random_calls(seed):
    """Batches of any kind: lengths, new tokens, heads, pages, windows, layouts and types drawn together."""
    r = random.Random(seed)
    B, Hkv, D, page = r.choice([1, 2, 5, 17, 40]), r.choice([1, 2, 3, 8]), r.choice([64, 128]), r.choice([8, 16, 64, 128, 512])
    H = Hkv * r.choice([1, 2, 3, 4, 7, 8, 20])
    lens = [r.choice([0, 1, 127, 128, 129, r.randint(1, 700), r.randint(1, 2500)]) for _ in range(B)]
    packed, kind = r.random() < 0.6, r.choice(["one", "few", "many"])
    most = {"one": 1, "few": 6, "many": 90}[kind]
    n = r.randint(1, most)
    news = [r.choice([0, 1, 1, r.randint(1, most)]) for _ in range(B)] if packed else [n] * B
    if sum(news) == 0:
        news[0] = 1
    causal = r.random() < 0.85
    window = r.choice([None, None, 1, 63, 500, 1500]) if causal else None
    run_attention(lens, news, H, Hkv, D, page, r.choice([torch.bfloat16, torch.float16]), r.random() < 0.5, packed=packed, seed=seed, hnd=r.random() < 0.7,
                  pad=r.choice([0, 0, 3, 200]) if packed else 0, causal=causal, window=window)
