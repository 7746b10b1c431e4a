"""What calls of rotary positions and of paged caches are refused for, without a GPU: the host side looks at the tensors before
anything is launched, so tensors of the CPU do."""

import pytest
import torch
from torch.autograd import forward_ad

from attn_engine import PagedKVCache, RotaryEmbedding
from core.native import lib


def pools(pages=4, page=16, heads=2, D=64, dtype=torch.bfloat16):
    return torch.zeros(pages, page, heads, D, dtype=dtype), torch.zeros(pages, page, heads, D, dtype=dtype)


def rotary(*args):
    """The native call behind RotaryEmbedding, with frequencies on the CPU."""
    host = lib.host()
    return host.rotary(host.make_turns(torch.zeros(32, dtype=torch.int64), 64, False, 1.0), *args)


def test_tangents_of_forward_mode_are_refused():
    """A dual tensor whose primal wants no gradient would come back without its tangent."""
    x, plain = torch.ones(2, 1, 2, 64), torch.ones(2, 1, 2, 64, dtype=torch.bfloat16)
    cache, table, lens = PagedKVCache(*pools()), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with forward_ad.dual_level():
        dual, dual16 = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(plain, torch.ones_like(plain))
        held = PagedKVCache(*(forward_ad.make_dual(t, torch.ones_like(t)) for t in pools()))
        calls = [lambda: rotary(dual, None, None, False), lambda: rotary(x, dual, None, False), lambda: rotary(dual, None, None, True),
                 lambda: rotary(dual[:, :, :1], None, None, False),   # a view of one
                 lambda: cache.attention(dual16, table, lens), lambda: cache.attention(plain, table, lens, out=dual16),
                 lambda: cache.append(dual16, plain, table, lens), lambda: cache.append(plain, dual16, table, lens),
                 lambda: held.attention(plain, table, lens), lambda: held.append(plain, plain, table, lens), lambda: held.read(table, lens, 4)]
        for call in calls:
            with pytest.raises(ValueError, match="forward"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="forward"):   # which does not turn forward mode off
                call()
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="CUDA"):   # the next refusal
            cache.attention(dual16, table, lens)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("which", ["k", "v", "k_scale", "v_scale"])
@pytest.mark.parametrize("how", ["data", "resized", "emptied", "shape"])
def test_pools_that_moved_are_refused(codes, which, how):
    """The native side knows where the pages were; it must not read there when they are not any more."""
    if not codes and "scale" in which:
        return
    kind = torch.float8_e4m3fn if codes else torch.bfloat16
    made = [torch.zeros(4, 16, 2, 64, dtype=kind) for _ in range(2)] + ([torch.zeros(4, 16, 2, dtype=torch.uint8) for _ in range(2)] if codes else [])
    cache, table, lens = PagedKVCache(*made), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    calls = [lambda: cache.read(table, lens, 4), lambda: cache.attention(q, table, lens), lambda: cache.append(q, q, table, lens)]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA"):   # the first refusal, as long as they are there
            call()
    pool = getattr(cache, which)
    if how == "data":
        pool.data = pool.clone()
    elif how == "resized":
        pool.resize_(8, *pool.shape[1:])
    elif how == "emptied":
        pool.untyped_storage().resize_(0)
    else:
        pool.data = pool.data.view(8, 8, *pool.shape[2:])
    for call in calls:
        with pytest.raises(ValueError, match="make a new one"):
            call()
    with pytest.raises(AttributeError):
        cache.k = made[0]


@pytest.mark.parametrize("codes", [False, True])
def test_one_pool_for_keys_and_values_is_not_written(codes):
    """Attention may read one pool as both; what an append left in it would be either."""
    kind, scale = (torch.float8_e4m3fn, torch.zeros(4, 16, 2, dtype=torch.uint8)) if codes else (torch.bfloat16, None)
    pool, other = (torch.zeros(4, 16, 2, 64, dtype=kind) for _ in range(2))
    table, lens, k = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    for cache in [PagedKVCache(pool, pool, scale, scale)] + ([PagedKVCache(pool, other, scale, scale)] if codes else []):
        with pytest.raises(ValueError, match="same memory"):
            cache.append(k, k, table, lens)
        with pytest.raises(ValueError, match="CUDA"):
            cache.attention(k, table, lens)


def test_frequencies_ask_their_own_device_for_a_capture(monkeypatch):
    """A call on a device that is not the current one: the capture that counts is under way there, or not at all."""
    current, capturing = [0], {1}

    class On:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] in capturing)
    with pytest.raises(lib.NativeError, match="before the capture"):
        RotaryEmbedding(8).native_on(torch.device("cuda", 1))
    assert current == [0]


def freed(*shape, dtype=torch.bfloat16):
    """A tensor whose storage was given back, as sharded training does between layers; not at the storage's begin."""
    t = torch.zeros(2, *shape, dtype=dtype)[1]
    t.untyped_storage().resize_(0)
    return t


def test_tensors_without_memory_are_refused():
    x, pos = torch.zeros(2, 1, 2, 64), torch.arange(1)
    calls = [lambda: rotary(freed(2, 1, 2, 64), None, None, False), lambda: rotary(x, freed(2, 1, 2, 64, dtype=torch.float32), None, False),
             lambda: rotary(x, None, freed(1, dtype=torch.int64), False), lambda: rotary(torch._efficientzerotensor(2, 1, 2, 64), None, pos, False),
             lambda: PagedKVCache(freed(4, 16, 2, 64), pools()[1]), lambda: PagedKVCache(pools()[0], freed(4, 16, 2, 64)),
             lambda: PagedKVCache(*pools(dtype=torch.float8_e4m3fn), torch.zeros(4, 16, 2, dtype=torch.uint8), freed(4, 16, 2, dtype=torch.uint8))]
    for call in calls:
        with pytest.raises(ValueError, match="no memory"):
            call()


def test_sizes_past_32_bits_are_refused():
    """4294967301 tokens are not 5: the launch counts in 32 bits."""
    row = torch.zeros(1, 1, 64)
    for q, k in ((row.expand(2 ** 32 + 5, 1, 64), None), (row.expand(1, 2 ** 32 + 5, 64), None), (row, row.expand(1, 2 ** 31, 64)),
                 (row.unsqueeze(0).expand(2 ** 31, 1, 1, 64), None)):
        with pytest.raises(ValueError, match="2\\^31"):
            rotary(q, k, None, False)
