"""Rotary positions and paged caches without a GPU: frequencies, what a call is refused for before anything is launched, the
oracle itself, and the argument structs."""

import copy
import math
import os
import pickle
import subprocess

import pytest
import torch

import metaattention_b200
from attn_engine import PagedKVCache, RotaryEmbedding
from attn_engine.rotary import rotary_frequencies
from core.native import lib
from examples_b200 import programs
from oracle import paged_math as pm


def test_public_names():
    assert metaattention_b200.PagedKVCache is PagedKVCache and metaattention_b200.RotaryEmbedding is RotaryEmbedding


# ---------------------------------------------------------------------------------------------------------------
# frequencies
# ---------------------------------------------------------------------------------------------------------------

def test_frequencies_plain_and_stretched():
    f, m = rotary_frequencies(8, 10000.0)
    assert m == 1.0 and f == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)
    assert rotary_frequencies(8, scaling="linear", factor=4.0)[0] == pytest.approx([x / 4 for x in f], rel=1e-15)
    g = rotary_frequencies(8, scaling="ntk", factor=16.0)[0]
    assert g[0] == 1.0 and g[-1] == pytest.approx(f[-1] / 16.0, rel=1e-12)   # the lowest is stretched by the factor
    y, m = rotary_frequencies(128, scaling="yarn", factor=16.0, original_length=4096)
    f = rotary_frequencies(128)[0]
    assert m == pytest.approx(0.1 * math.log(16.0) + 1.0)
    for i, (a, b) in enumerate(zip(y, f)):
        turns = 4096 * b / (2 * math.pi)
        if turns > 40:
            assert a == b, i
        if turns < 0.8:
            assert a == pytest.approx(b / 16.0, rel=1e-14), i
        assert b / 16.0 * (1 - 1e-14) <= a <= b


def test_turns_are_the_frequencies_as_fractions_of_a_turn():
    rope = RotaryEmbedding(64)
    for f, t in zip(rope.frequencies, rope.turns()):
        assert abs(t / 2.0 ** 64 - f / (2 * math.pi)) <= 2.0 ** -53
    # a far position: the wrapped 64-bit product against the angle with all digits
    from fractions import Fraction
    for f, t in zip(rope.frequencies, rope.turns()):
        pos = 1048573
        part = ((t * pos) % (1 << 64)) / 2.0 ** 64
        exact = float(Fraction(f) * pos / Fraction(2 * math.pi) % 1)
        assert abs((part - exact + 0.5) % 1.0 - 0.5) <= 1e-12


@pytest.mark.parametrize("args", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, scaling="other"),
                                  dict(rotary_dim=8, scaling="linear", factor=0.5), dict(rotary_dim=8, factor=math.inf), dict(rotary_dim=2, scaling="ntk"),
                                  dict(rotary_dim=8, frequencies=[1.0] * 3), dict(rotary_dim=2, frequencies=[math.nan]), dict(rotary_dim=8, magnitude=math.nan),
                                  dict(rotary_dim=8, scaling="yarn", beta_fast=1.0, beta_slow=2.0)])
def test_frequencies_refused(args):
    with pytest.raises(ValueError):
        RotaryEmbedding(**args)


def test_rotary_needs_a_gpu():
    with pytest.raises(lib.NativeError):
        RotaryEmbedding(8)(torch.zeros(1, 2, 8, dtype=torch.bfloat16))


def test_rotary_copies_and_pickles():
    rope = RotaryEmbedding(16, interleaved=True, scaling="linear", factor=2.0)
    for other in (copy.deepcopy(rope), pickle.loads(pickle.dumps(rope))):
        assert other.frequencies == rope.frequencies and other.interleaved and other.turns() == rope.turns()


# ---------------------------------------------------------------------------------------------------------------
# refusals (the host side looks at shapes, types, strides and devices, so tensors of the CPU do)
# ---------------------------------------------------------------------------------------------------------------

def pools(pages=4, page=16, heads=2, D=64, dtype=torch.bfloat16):
    return torch.zeros(pages, page, heads, D, dtype=dtype), torch.zeros(pages, page, heads, D, dtype=dtype)


def scales(pages=4, page=16, heads=2, dtype=torch.uint8):
    return torch.zeros(pages, page, heads, dtype=dtype), torch.zeros(pages, page, heads, dtype=dtype)


@pytest.mark.parametrize("make,word", [
    (lambda: PagedKVCache(torch.zeros(4, 16, 64, dtype=torch.bfloat16), torch.zeros(4, 16, 64, dtype=torch.bfloat16)), "num_pages"),
    (lambda: PagedKVCache(pools()[0], pools(pages=5)[0]), "same shape"),
    (lambda: PagedKVCache(pools()[0], pools(dtype=torch.float16)[0]), "dtype"),
    (lambda: PagedKVCache(*pools(dtype=torch.float32)), "float8_e4m3fn"),
    (lambda: PagedKVCache(*pools(D=96)), "head_dim"),
    (lambda: PagedKVCache(*pools(page=24)), "page_size"),
    (lambda: PagedKVCache(*pools(page=4)), "page_size"),
    (lambda: PagedKVCache(*pools(pages=0)), "empty"),
    (lambda: PagedKVCache(*pools(), *scales()), "scale"),
    (lambda: PagedKVCache(*pools(dtype=torch.float8_e4m3fn)), "scale"),
    (lambda: PagedKVCache(*pools(dtype=torch.float8_e4m3fn), *scales(dtype=torch.float32)), "e8m0"),
    (lambda: PagedKVCache(*pools(dtype=torch.float8_e4m3fn), *scales(page=8)), "scales must be"),
    (lambda: PagedKVCache(*(torch.zeros(4, 16, 2, 66, dtype=torch.bfloat16)[..., 1:65] for _ in range(2))), "16 bytes"),
    (lambda: PagedKVCache(*(torch.zeros(4, 16, 64, 2, dtype=torch.bfloat16).transpose(2, 3) for _ in range(2))), "contiguous"),
    (lambda: PagedKVCache(*(torch.zeros(4, 16, 1, 64, dtype=torch.bfloat16).expand(4, 16, 2, 64) for _ in range(2))), "positive"),
])
def test_pools_refused(make, word):
    with pytest.raises(ValueError, match=word):
        make()


def test_calls_on_the_cpu_are_refused():
    cache = PagedKVCache(*pools())
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: cache.append(k, k, table, lens), lambda: cache.read(table, lens, 4), lambda: cache.attention(k, table, lens)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_caches_copy_and_pickle():
    cache = PagedKVCache.allocate(4, 16, 2, 64, dtype=torch.float8_e4m3fn, device="cpu")
    assert cache.k.shape == (4, 16, 2, 64) and cache.k_scale.shape == (4, 16, 2) and cache.k_scale.dtype == torch.float8_e8m0fnu
    cache.k.view(torch.uint8)[1, 2, 1] = 5
    other = copy.deepcopy(cache)
    assert torch.equal(other.k.view(torch.uint8), cache.k.view(torch.uint8)) and other.k.data_ptr() != cache.k.data_ptr() and other._native is not cache._native


# ---------------------------------------------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("top,e", [(448.0, 0), (448.0001, 1), (1.75, -8), (1.7500001, -7), (2.0 ** -133, -127), (3.3e38, 120), (0.0, -127)])
def test_exponent(top, e):
    assert pm.exponent_of(top) == e


def test_codes_are_the_nearest():
    row = torch.randn(64, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    codes, byte = pm.quantise(row)
    back = codes.double() * 2.0 ** (byte - 127)
    # half a step of a 3-bit mantissa, or of the least subnormal
    assert ((back - row).abs() <= torch.maximum(row.abs() * 2.0 ** -4, torch.tensor(2.0 ** (byte - 127 - 10)))).all()


def test_oracle_attention_matches_a_dense_softmax():
    g = torch.Generator().manual_seed(4)
    q, k, v = torch.randn(5, 4, 8, generator=g).double(), torch.randn(12, 2, 8, generator=g).double(), torch.randn(12, 2, 8, generator=g).double()
    o, lse, _ = pm.attention(q, k, v, 12, 5, 0.3, window=6)
    s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(2, 1)) * 0.3
    i, j = torch.arange(7, 12).view(-1, 1), torch.arange(12)
    s = s.masked_fill(~((j <= i) & (j > i - 6)), -math.inf)
    assert torch.allclose(lse, s.logsumexp(2)) and torch.allclose(o, torch.einsum("hij,jhd->ihd", s.softmax(2), v.repeat_interleave(2, 1)))


# ---------------------------------------------------------------------------------------------------------------
# C ABI
# ---------------------------------------------------------------------------------------------------------------

def test_struct_layouts_match_header(tmp_path):
    probes = {
        "AttnB200Rotary": (lib.Rotary, ["dim", "magnitude"]),
        "AttnB200RotaryArgs": (lib.RotaryArgs, ["y", "positions", "y_stride", "pos_stride", "heads", "dtype", "inverse", "rotary"]),
        "AttnB200PagedCache": (lib.PagedCacheArgs, ["k_scale", "v_stride", "v_scale_stride", "block_table", "seq_lens", "num_pages", "dtype"]),
        "AttnB200PagedAppendArgs": (lib.PagedAppendArgs, ["k", "cu_seqlens", "v_stride", "seq", "rotary"]),
        "AttnB200PagedReadArgs": (lib.PagedReadArgs, ["v", "max_len", "dtype"]),
        "AttnB200PagedAttnArgs": (lib.PagedAttnArgs, ["q", "lse", "o_stride", "heads", "scale", "window", "workspace_bytes"]),
    }
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "attn_b200.h"', "int main(void) {"]
    for name, (_, fields) in probes.items():
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f in fields]
    (tmp_path / "probe.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-I", lib.INCLUDE_DIR, "-o", str(tmp_path / "probe"), str(tmp_path / "probe.c")], check=True)
    seen = dict(x.split() for x in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, (mirror, fields) in probes.items():
        import ctypes
        assert int(seen[name]) == ctypes.sizeof(mirror), name
        for f in fields:
            assert int(seen[f"{name}.{f}"]) == getattr(mirror, f).offset, f"{name}.{f}"


def test_null_arguments_are_refused_without_a_gpu(native_lib):
    assert native_lib.attn_b200_rotary(None, None) == -1
    assert native_lib.attn_b200_paged_append(None, None) == -1
    assert native_lib.attn_b200_paged_read(None, None) == -1
    assert native_lib.attn_b200_paged_attention(None, None) == -1
    assert native_lib.attn_b200_paged_workspace_bytes(None) == -1
    import ctypes
    assert native_lib.attn_b200_paged_attention(ctypes.byref(lib.PagedAttnArgs()), None) == -1


# ---------------------------------------------------------------------------------------------------------------
# an engine's program over a cache
# ---------------------------------------------------------------------------------------------------------------

class Recorder:
    """Takes the place of a cache and keeps what it is asked."""

    def attention(self, q, *args, **kwargs):
        self.args, self.kwargs = args, kwargs
        return "o", "lse"


@pytest.mark.parametrize("mask,causal,window", [(None, False, None), (programs.causal, True, None), (programs.sliding_window_mask, True, 128)])
def test_an_engine_gives_its_scale_and_mask_to_a_cache(mask, causal, window):
    eng, cache = programs.masked_softmax_engine(1, 2, 300, 64, 64, mask), Recorder()
    q = torch.zeros(1, 1, 2, 64, dtype=eng.dtype)
    assert eng.paged_attention(q, cache, "table", "lens", out="out") == "o"
    assert cache.args == ("table", "lens", None) and cache.kwargs.pop("scale") == pytest.approx(0.125, rel=1e-6)
    assert cache.kwargs == {"causal": causal, "window": window, "out": "out", "return_lse": True}
    assert list(eng.last_final_rowscales.values()) == ["lse"]


def test_engines_whose_programs_a_cache_does_not_run():
    q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    engines = [programs.masked_softmax_engine(1, 2, 300, 64, 64, lambda b, h, i, j: (i - j < 9) & (j - i < 9)),      # looks ahead
               programs.masked_softmax_engine(1, 2, 300, 64, 64, lambda b, h, i, j: j >= i),
               programs.masked_softmax_engine(1, 2, 300, 64, 64, lambda b, h, i, j: (j <= i) & (i // 7 == j // 7)),
               programs.sparse_decode_engine(1, 2, 2, 300, 64, 64)]
    for eng in engines:
        with pytest.raises(NotImplementedError, match="paged"):
            eng.paged_attention(q, Recorder(), None, None)
    eng = programs.masked_softmax_engine(1, 2, 300, 64, 64, None)
    with pytest.raises(TypeError, match="float16"):
        eng.paged_attention(q.half(), Recorder(), None, None)
