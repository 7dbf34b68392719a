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
    -> (out, lse, sum of p |v|: what weights rounded on the way are measured by)"""
    n, heads, dim = q.shape
    n_blocks, _, kv_heads, _ = keys.shape
    group = heads // kv_heads
    out, lse, mass = np.zeros((n, heads, dim)), np.full((n, heads), -np.inf), np.zeros((n, heads, dim))
    for b in range(n):
        length = max(0, min(int(lens[b]), tables.shape[1] * block))
        t = np.arange(max(0, length - window) if window else 0, length)
        if t.size == 0:
            continue
        page = tables[b][t // block].astype(np.int64)
        t, page = t[(page >= 0) & (page < n_blocks)], page[(page >= 0) & (page < n_blocks)]
        if t.size == 0:
            continue
        k, v = keys[page, t % block] * k_scale, values[page, t % block] * v_scale
        for h in range(heads):
            z = scale * (k[:, h // group] @ q[b, h])
            if cap:
                z = cap * np.tanh(z / cap)
            top = z.max()
            with np.errstate(invalid="ignore"):
                p = np.exp(z - top)
            lse[b, h] = top + np.log(p.sum())
            p = p / p.sum()
            out[b, h] = p @ v[:, h // group]
            mass[b, h] = p @ np.abs(v[:, h // group])
    return out, lse, mass
