"""Definitions of the paged 8-bit cache operators in 64 bits on the CPU (loops, no cleverness)."""

from __future__ import annotations

import math

import numpy as np
import torch

BLOCK = 32


def e4m3_values() -> np.ndarray:
    """Value of each of the 256 E4M3 codes."""
    out = np.zeros(256)
    for code in range(256):
        sign, field, fraction = code >> 7, (code >> 3) & 15, code & 7
        value = math.ldexp(1 + fraction / 8, field - 7) if field else math.ldexp(fraction / 8, -6)
        out[code] = math.nan if code & 127 == 127 else (-value if sign else value)
    return out


VALUES = e4m3_values()
_FINITE = VALUES[:127]  # 0 .. 448, ascending


def encode(x: np.ndarray) -> np.ndarray:
    """Nearest code (ties to the even code), saturating; NaN -> 0x7f with the sign kept free."""
    x = np.asarray(x, np.float64)
    mag = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), 448.0)
    hi = np.clip(np.searchsorted(_FINITE, mag), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _FINITE[hi] - mag, mag - _FINITE[lo]
    code = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    code = np.where(np.signbit(x), code | 128, code)
    return np.where(np.isnan(x), 127, code).astype(np.uint8)


def needed_scale(top: float) -> int:
    """Code of the smallest power of two that takes ``top`` to 448 or less, at least 2^-99."""
    code = 28
    while top > math.ldexp(448.0, code - 127):
        code += 1
    return code


def write(values, scales, rows, table, seq_lens, cu, pages, page):
    """``values`` uint8 [pages, H, page, D], ``scales`` uint8 [pages, H, page/32] (numpy, in
    place); ``rows`` float64 [T, H, D]."""
    batch = len(seq_lens)
    cu = list(range(batch + 1)) if cu is None else cu
    heads = values.shape[1]
    for b in range(batch):
        n = cu[b + 1] - cu[b]
        start = seq_lens[b] - n
        position = max(start, 0)
        while position < seq_lens[b]:
            end = min(seq_lens[b], (position // BLOCK + 1) * BLOCK)
            if position // page >= table.shape[1]:
                break
            at = int(table[b, position // page])
            if 0 <= at < pages:
                block, kept = position % page // BLOCK, position % BLOCK
                for h in range(heads):
                    new = rows[cu[b] + position - start : cu[b] + end - start, h]
                    finite = np.abs(new[np.isfinite(new)])
                    code = needed_scale(float(finite.max()) if finite.size else 0.0)
                    lo = block * BLOCK
                    if kept:
                        old = int(scales[at, h, block])
                        code = max(code, old)
                        if code > old:
                            held = VALUES[values[at, h, lo : lo + kept]] * 2.0 ** (old - code)
                            values[at, h, lo : lo + kept] = encode(held)
                    values[at, h, lo + kept : lo + kept + end - position] = encode(
                        new * 2.0 ** (127 - code))
                    scales[at, h, block] = code
            position = end


def read(values, scales, table, positions_of):
    """float64 [H, D] rows of ``positions_of`` = list of (sequence, position)."""
    pages, heads, page, dim = values.shape
    out = np.zeros((len(positions_of), heads, dim))
    for i, (b, position) in enumerate(positions_of):
        if position < 0 or position // page >= table.shape[1]:
            continue
        at = int(table[b, position // page])
        if 0 <= at < pages:
            scale = 2.0 ** (scales[at, :, position % page // BLOCK].astype(np.float64) - 127)
            out[i] = VALUES[values[at, :, position % page]] * scale[:, None]
    return out


def named(table, b, position, pages, page):
    """Whether the block table names a page for the position."""
    return position // page < table.shape[1] and 0 <= int(table[b, position // page]) < pages


def attention(q, k_values, v_values, k_scales, v_scales, table, seq_lens, cu, scale, causal):
    """``q`` float64 [T, Hq, D] -> float64 [T, Hq, D]; rows that see nothing are zero."""
    pages, heads, page, dim = k_values.shape
    batch = len(seq_lens)
    cu = list(range(batch + 1)) if cu is None else cu
    group = q.shape[1] // heads
    out = np.zeros(q.shape)
    for b in range(batch):
        length = min(int(seq_lens[b]), table.shape[1] * page)
        where = [(b, p) for p in range(length)]
        seen = np.array([named(table, b, p, pages, page) for p in range(length)], bool)
        k = read(k_values, k_scales, table, where)
        v = read(v_values, v_scales, table, where)
        n = cu[b + 1] - cu[b]
        for i in range(n):
            position = int(seq_lens[b]) - n + i
            allowed = seen & (np.arange(length) <= position) if causal else seen
            if not allowed.any():
                continue
            for h in range(q.shape[1]):
                s = k[allowed, h // group] @ q[cu[b] + i, h] * scale
                w = np.exp(s - s.max())
                out[cu[b] + i, h] = (w[:, None] * v[allowed, h // group]).sum(0) / w.sum()
    return out


def rotary(x, positions, inv_freq, axis, adjacent=False):
    """``x`` float64 [T, H, D]; ``positions`` [axes, T]."""
    half = len(inv_freq)
    y = np.array(x, np.float64)
    angle = positions[axis].T.astype(np.float64) * inv_freq
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a = slice(0, 2 * half, 2) if adjacent else slice(0, half)
    b = slice(1, 2 * half, 2) if adjacent else slice(half, 2 * half)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def to_numpy(tensor: torch.Tensor) -> np.ndarray:
    return tensor.detach().cpu().double().numpy()
