"""Plain 64-bit forms of the operators on the paged cache, in numpy on the CPU, and what their
tests share. Tolerances count roundings: one to type t is off by at most half a step, eps(t) / 2
relative to the value (or half the smallest subnormal step), one operation in 32 bits by 2^-24."""
import numpy as np

from kvt_amd import ctypes_defs

SHAPES = {"flash": ctypes_defs.SHAPE_FLASH, "ragged": ctypes_defs.SHAPE_RAGGED_FLASH,
          "hnd": ctypes_defs.SHAPE_FLASHINFER, "pages": ctypes_defs.SHAPE_QWEN3_NEXT_FLASH}
# half a step, torch.finfo(t).eps / 2: relative to the value, and absolute below the normal numbers
HALF_STEP = {"bf16": (2.0 ** -8, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "f32": (2.0 ** -24, 0.0),
             "e4m3": (2.0 ** -4, 2.0 ** -10)}


def torch_type(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
            "e4m3": torch.float8_e4m3fn}[name]


def cache_shape(layout, n_blocks, block, heads, dim):
    return {"flash": (2, n_blocks, block, heads, dim), "ragged": (n_blocks, block, 2, heads, dim),
            "hnd": (n_blocks, 2, heads, block, dim), "pages": (n_blocks, 2, block, heads, dim)}[layout]


def kv_views(layout, cache):
    """(keys, values) as [n_blocks, block, heads, dim] views of a torch tensor or numpy array."""
    if layout == "flash":
        return cache[0], cache[1]
    if layout == "ragged":
        return cache[:, :, 0], cache[:, :, 1]
    k, v = cache[:, 0], cache[:, 1]
    if layout == "hnd":
        return (k.swapaxes(1, 2), v.swapaxes(1, 2))
    return k, v


def wide(t):
    """A torch tensor of any of the types as float64 numpy."""
    import torch
    return t.detach().to(torch.float32 if t.dtype != torch.float64 else torch.float64).cpu().numpy().astype(np.float64)


def rotated(x, positions, freq, magnitude, rotary_dim, interleaved):
    """-> (rotated rows, per element |x0| + |x1| of its pair: what 32-bit rounding is measured by)"""
    y, scale = x.copy(), np.abs(x)
    angle = positions.astype(np.float64)[:, None, None] * np.asarray(freq)
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle)
    h = rotary_dim // 2
    i0, i1 = (slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if interleaved else (slice(0, h), slice(h, rotary_dim))
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    scale[..., i0] = scale[..., i1] = abs(magnitude) * (np.abs(a) + np.abs(b))
    return y, scale


def rotation_tolerance(exact, scale, kind):
    """One rounding to the output's type, and 32 bits on the way: the cosine and sine from an angle
    rounded to 32 bits after its reduction to an eighth of a turn (2^-24 * pi / 4 and two units of
    the function, times the magnitude: under 4 roundings), two products, a sum: 8 roundings of
    2^-24 of |x0| + |x1|."""
    rel, floor = HALF_STEP[kind]
    return rel * np.abs(exact) * (1 + 2.0 ** -10) + floor + 8 * 2.0 ** -24 * scale


def decode_exact(q, keys, values, tables, lens, block, scale, window=0, cap=0.0, k_scale=1.0, v_scale=1.0):
    """Attention of one token per sequence in 64 bits: q [seqs, heads, dim], keys / values
    [n_blocks, block, kv_heads, dim] as float64; a page outside the cache is not seen.
    -> (out, lse, measure), measure = what decode_tolerance() goes by, per (sequence, head): the
    sum of p |v| for every dim, the largest sum of |q k| of a score, tokens seen, the largest |v|."""
    n, heads, dim = q.shape
    n_blocks, _, kv_heads, _ = keys.shape
    group = heads // kv_heads
    out, lse = np.zeros((n, heads, dim)), np.full((n, heads), -np.inf)
    mass, size, count, most = np.zeros((n, heads, dim)), np.zeros((n, heads)), np.zeros((n, heads)), np.zeros((n, heads))
    for b in range(n):
        length = max(0, min(int(lens[b]), tables.shape[1] * block))
        t = np.arange(max(0, length - window) if window else 0, length)
        if t.size == 0:
            continue
        page = tables[b][t // block].astype(np.int64)
        held = (page >= 0) & (page < n_blocks)
        t, page = t[held], page[held]
        if t.size == 0:
            continue
        k, v = keys[page, t % block] * k_scale, values[page, t % block] * v_scale
        for h in range(heads):
            z = scale * (k[:, h // group] @ q[b, h])
            if cap:
                z = cap * np.tanh(z / cap)
            top = z.max()
            p = np.exp(z - top)
            lse[b, h] = top + np.log(p.sum())
            p = p / p.sum()
            out[b, h], mass[b, h] = p @ v[:, h // group], p @ np.abs(v[:, h // group])
            size[b, h] = abs(scale) * (np.abs(k[:, h // group]) @ np.abs(q[b, h])).max()
            count[b, h], most[b, h] = t.size, np.abs(v[:, h // group]).max()
    return out, lse, (mass, size, count, most)


def decode_tolerance(out, lse, measure, kind):
    """(of out, of lse). In 32 bits a score is off by (dim + 8) 2^-24 of the sum of its |q k|: dim
    additions, the scale, the change of base and the difference to the maximum (the products of two
    16-bit values are exact); the weights of a softmax by twice that, relative, and 4 roundings of
    the exponential. Sums over n tokens: n roundings of 2^-24 of the sum of p |v|. A weight in two
    16-bit values, cut off (a step, 2^-7 for bf16 and 2^-10 for f16) and the rest rounded (half a
    step): 2^-15 or 2^-21 of it; the rest is at least the smallest positive number, for f16 (2^-24, of
    weights times 2^15) 2^-39 of every |v|, and rounded by half of that. Joining parts and dividing: 8 more. Then the output's own rounding."""
    mass, size, count, most = measure
    dim = out.shape[-1]
    score = (dim + 8) * 2.0 ** -24 * size
    split = 2.0 ** -15 if kind == "bf16" else 2.0 ** -21
    rel = 2 * score + (12 + count) * 2.0 ** -24 + split
    tol = rel[..., None] * mass + (0 if kind == "bf16" else 1.5 * 2.0 ** -39 * (count * most)[..., None])
    half, floor = HALF_STEP[kind]
    seen = np.isfinite(lse)
    return (half * (np.abs(out) + tol) + floor + tol,
            score + (16 + count + 2 * np.where(seen, np.abs(lse), 0) + 2 * size) * 2.0 ** -24)
