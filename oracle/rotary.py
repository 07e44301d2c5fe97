"""Rotary positions, appends into a paged cache and its reading back, from their definitions on
the CPU: rotations in float64, block by block and row by row in order."""

import math

import torch

FLT_MIN = 2.0 ** -126
TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def rotate(x, positions, turns, amplitude=1.0, interleaved=False, inverse=False):
    """x [rows, heads, dim] float64: pair p as a complex number times amplitude e^(+-i angle)."""
    y = x.double().clone()
    r = 2 * turns.shape[0]
    # whole turns off before the sine: exact in float64 up to the product's own rounding
    t = positions.double()[:, None] * turns.double()
    angle = (t - t.round()) * (2 * math.pi) * (-1 if inverse else 1)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(y[..., a], y[..., b]) * torch.polar(torch.full_like(angle, amplitude), angle)[:, None]
    y[..., a], y[..., b] = z.real, z.imag
    return y


def rotate_error(x, turns, amplitude=1.0, interleaved=False):
    """How far float32 may be from ``rotate``, per element: sines and cosines within 2^-23, times
    the amplitude (one rounding, 2^-24), two products and a sum (2^-24 each): (|a| + |b|) times
    amplitude 2^-23 (1 + 1/2 + 1/2 + 1/2), taken as 2^-21."""
    x = x.double().abs()
    r = 2 * turns.shape[0]
    e = torch.zeros_like(x)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    both = (x[..., a] + x[..., b]) * abs(amplitude) * 2.0 ** -21
    e[..., a], e[..., b] = both, both
    return e


def codes_of(x, scale, dtype):
    """float32 x over its scale as codes: IEEE division, clamped, to the nearest even."""
    y = x.float() / scale
    if dtype == torch.int8:
        return torch.where(y.isnan(), torch.zeros(()), y.clamp(-127, 127).round()).to(torch.int8)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn)


def block_scale(x, dtype):
    """Scale of the rows x [rows, heads, dim] of one block, per head."""
    a = x.float().abs()
    a = torch.where(a.isfinite(), a, torch.zeros(()))
    return (a.amax(dim=(0, 2)) * torch.tensor(1.0 / TOP[dtype], dtype=torch.float32)).clamp_min(FLT_MIN)


def append(cache, scale, rows, tables, lengths, counts):
    """Rows (float32) appended in place, sequence after sequence; scale None (a pool of a row
    type), 0-d, [block, token, head] or [block, head]."""
    bs = cache.shape[1]
    begin = 0
    for s, (length, n) in enumerate(zip(lengths, counts)):
        places = []
        for i in range(n):
            pos = length - n + i
            block = int(tables[s, pos // bs]) if 0 <= pos < tables.shape[1] * bs else -1
            if 0 <= block < cache.shape[0]:
                places.append((block, pos % bs, begin + i))
        if scale is None:
            for block, o, r in places:
                cache[block, o] = rows[r].to(cache.dtype)
        elif scale.ndim != 2:
            for block, o, r in places:
                if scale.ndim == 0:
                    f = scale
                else:
                    f = (rows[r].float().abs().amax(-1) * torch.tensor(1 / 448, dtype=torch.float32))
                    f = torch.where(f < FLT_MIN, torch.tensor(FLT_MIN), f)
                    scale[block, o] = f
                    f = f[:, None]
                cache[block, o] = codes_of(rows[r], f, cache.dtype)
        else:
            while places:
                block, o = places[0][:2]
                here = [p for p in places if p[0] == block]
                places = [p for p in places if p[0] != block]
                new = rows[[p[2] for p in here]]
                f, old = block_scale(new, cache.dtype), scale[block].clone()
                if o:
                    f = torch.where(old > f, old, f)
                    grew = (f > old)[:, None]
                    again = codes_of(cache[block, :o].float() * old[:, None], f[:, None], cache.dtype)
                    cache[block, :o] = torch.where(grew, again.float(), cache[block, :o].float()).to(cache.dtype)
                scale[block] = f
                cache[block, o:o + len(here)] = codes_of(new, f[:, None], cache.dtype)
        begin += n


def load(cache, scale, tables, lengths, counts):
    """The last counts[s] positions of every sequence as float64; zeros where nothing is held."""
    bs = cache.shape[1]
    out = []
    for s, (length, n) in enumerate(zip(lengths, counts)):
        for i in range(n):
            pos = length - n + i
            block = int(tables[s, pos // bs]) if 0 <= pos < tables.shape[1] * bs else -1
            x = torch.zeros(cache.shape[2:], dtype=torch.float64)
            if 0 <= block < cache.shape[0]:
                x = cache[block, pos % bs].float().double()
                if scale is not None:
                    f = scale if scale.ndim == 0 else (
                        scale[block] if scale.ndim == 2 else scale[block, pos % bs])[:, None]
                    x = x * f.double()
            out.append(x)
    return torch.stack(out) if out else torch.zeros((0, *cache.shape[2:]), dtype=torch.float64)


def dequantized(cache, scale):
    """The whole pool as float64 numbers."""
    f = scale.double()
    return cache.float().double() * (f if f.ndim == 0 else f[:, None, :, None] if f.ndim == 2
                                     else f[..., None])
