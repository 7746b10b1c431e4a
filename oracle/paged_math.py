"""Plain restatement of the operators around a paged cache, on the CPU in 64 bits and token by token: rotary positions, codes and
scales of an 8-bit row, writing, reading back and attention.  TEST INFRASTRUCTURE (see reference_math.py)."""

from __future__ import annotations

import math

import torch


def rotary(x, positions, frequencies, magnitude=1.0, interleaved=False, sign=1.0):
    """x [..., heads, D] with positions [...]: pair i of the first 2 * len(frequencies) columns turned by sign * position * f_i."""
    y = x.double().clone()
    n = len(frequencies)
    angle = sign * positions.double().unsqueeze(-1) * torch.tensor(frequencies, dtype=torch.float64)
    c, s = (angle.cos() * magnitude).unsqueeze(-2), (angle.sin() * magnitude).unsqueeze(-2)
    first = torch.arange(n) * 2 if interleaved else torch.arange(n)
    second = first + (1 if interleaved else n)
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first] = a * c - b * s
    y[..., second] = b * c + a * s
    return y


def exponent_of(top: float) -> int:
    """The least e >= -127 with top <= 448 * 2^e."""
    if top == 0:
        return -127
    m, x = math.frexp(top)
    return max(-127, x - 9 if m <= 0.875 else x - 8)


def quantise(row):
    """(codes float8_e4m3fn [D], exponent byte) of one row."""
    row = row.double()
    if not bool(torch.isfinite(row).all()):
        return torch.full(row.shape, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn), 255
    e = exponent_of(float(row.abs().max()))
    return (row * 2.0 ** -e).float().to(torch.float8_e4m3fn), e + 127   # exact in 32 bits: a power of two


def values(pool, scale, page, row, head):
    """The row's values in 64 bits; None where the page does not exist (reads as zeros)."""
    if page < 0 or page >= pool.shape[0]:
        return None
    x = pool[page, row, head]
    if scale is None:
        return x.double()
    byte = int(scale.view(torch.uint8)[page, row, head])
    return x.float().double() * (float("nan") if byte == 255 else 2.0 ** (byte - 127))


def sequence(pool, scale, table_row, length):
    """[length, heads, D] in 64 bits; zeros where a page does not exist."""
    page_size, heads, D = pool.shape[1], pool.shape[2], pool.shape[3]
    out = torch.zeros(length, heads, D, dtype=torch.float64)
    for t in range(length):
        for h in range(heads):
            x = values(pool, scale, int(table_row[t // page_size]), t % page_size, h)
            if x is not None:
                out[t, h] = x
    return out


def rows_of(cu, seq, batch):
    """(first row, rows) of every sequence's new tokens; batched calls: rows of the flattened [batch * seq]."""
    if cu is None:
        return [(b * seq, seq) for b in range(batch)]
    return [(int(cu[b]), int(cu[b + 1] - cu[b])) for b in range(batch)]


def attention(q, k, v, length, fresh, scale, causal=True, window=None):
    """q [fresh, H, D] at the last positions of a sequence with k, v [length, Hkv, D]: (o, lse [H, fresh], A), A the sum of the
    magnitudes that went into each output."""
    H, G = q.shape[1], q.shape[1] // k.shape[1]
    pos = torch.arange(length - fresh, length).unsqueeze(1)
    at = torch.arange(length).unsqueeze(0)
    keep = (at <= pos) & (pos >= 0) if causal else torch.ones(fresh, length, dtype=torch.bool)
    if window is not None:
        keep &= at > pos - window
    o, mag, lse = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), torch.full((H, fresh), -math.inf, dtype=torch.float64)
    for h in range(H):
        for i in range(fresh):
            which = keep[i].nonzero().flatten()
            if which.numel() == 0:
                continue
            s = k[which, h // G] @ q[i, h].double() * scale
            lse[h, i] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[h, i])
            o[i, h] = p @ v[which, h // G]
            mag[i, h] = p @ v[which, h // G].abs()
    return o, lse, mag
