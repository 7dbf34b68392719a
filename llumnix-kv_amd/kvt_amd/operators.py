"""The operators on the registered cache (include/kvt_hip.h, "operators on the registered cache"):
rotary positions, the append of a step's keys and values to its pages, and the attention of one new
token over them.

Tensors are torch tensors on the cache's device (any strides; the elements of a row next to each
other), `stream` a hipStream_t handle as everywhere in this package (None: the default stream).
Sizes, types and devices are checked here, everything else by the library."""
import ctypes as C

from .binding import KvLayoutStruct, KvtError, RotaryOpts, _quiet_close, check, lib
from .ctypes_defs import ERR_INVALID

DTYPES = {"bf16": 0, "f16": 1, "f32": 2, "e4m3": 3}
SCALINGS = {"plain": 0, "linear": 1, "bands": 2, "ramp": 3}
_types = {}          # "int32", "int64" and the codes above -> torch dtype; torch dtype -> code


def _torch_types():
    """Made by the first call that is given a tensor (this package does without torch), and put in place
    whole: another thread finds all of it or nothing."""
    global _types
    import torch
    named = {0: torch.bfloat16, 1: torch.float16, 2: torch.float32}
    _types = {**named, **{t: code for code, t in named.items()}, "int32": torch.int32, "int64": torch.int64}
    return _types


def _code(tensor, name):
    code = (_types or _torch_types()).get(tensor.dtype)
    if code is None:
        raise ValueError("%s: unsupported type %s" % (name, tensor.dtype))
    return code


def _rows(tensor, name, shape, code):
    """(pointer, token stride, head stride) in bytes of a [tokens, heads, dim] tensor."""
    if tensor.shape != shape or tensor.dtype != _types[code]:
        raise ValueError("%s: got %s of %s, expected %s of %s" % (name, tuple(tensor.shape), tensor.dtype, shape,
                                                                  _types[code]))
    t, h, e = tensor.stride()
    if e != 1 and shape[2] > 1:
        raise ValueError("%s: the elements of a row must lie next to each other" % name)
    size = 4 if code == 2 else 2
    return tensor.data_ptr(), t * size, h * size


def _index(tensor, name, shape, kind):
    """Pointer of a contiguous tensor of one type ("int32", "int64" or a code)."""
    if tensor.shape != shape or tensor.dtype != _types[kind] or not tensor.is_contiguous():
        raise ValueError("%s: expected a contiguous %s tensor of shape %s" % (name, _types[kind], shape))
    return tensor.data_ptr()


def _refuse_elsewhere(device, tensors):
    """Refuses tensors that the device's kernels may not reach: those of another device, or in plain host
    memory. (The library sees pointers, and inside a capture does not ask the runtime about them.)"""
    for name, t in tensors.items():
        if t is not None and t.get_device() != device and not (t.get_device() < 0 and t.is_pinned()):
            raise KvtError(ERR_INVALID, "%s and what it is used with are not on one device (%d)" % (name, device))


class KvLayout:
    """Where the rows of a cache lie (kvt_kv_layout): a dense cache of one of the cache shapes, or
    with `strides` = (block, kv, token, head) in bytes any other. dtype: "bf16", "f16", "e4m3"."""

    def __init__(self, cache_shape, dtype, n_blocks, tokens_per_block, n_kv_heads, head_dim, tensor=0,
                 strides=None):
        s = KvLayoutStruct()
        if strides is None:
            check(lib().kvt_kv_layout_of(cache_shape, DTYPES[dtype], n_blocks, tokens_per_block, n_kv_heads,
                                         head_dim, C.byref(s)))
            s.tensor = tensor
        else:
            s = KvLayoutStruct(DTYPES[dtype], tensor, n_kv_heads, head_dim, tokens_per_block, 0, n_blocks, *strides)
        self.struct, self.n_kv_heads, self.head_dim = s, n_kv_heads, head_dim
        self.ref = C.byref(s)


def rotary_frequencies(rotary_dim, base=10000.0, scaling="plain", factor=1.0, original_max_position=0, low=0.0,
                       high=0.0, magnitude=0.0):
    """-> (radians per position of every pair, what rotated values are multiplied with);
    see kvt_rotary_frequencies."""
    freq, mag = (C.c_double * max(1, rotary_dim // 2))(), C.c_double()
    opts = RotaryOpts(rotary_dim, SCALINGS[scaling], base, factor, original_max_position, low, high, magnitude)
    check(lib().kvt_rotary_frequencies(C.byref(opts), freq, C.byref(mag)))
    return list(freq), mag.value


class Rotary:
    """A rotation of the first rotary_dim elements of a row by its position (kvt_rotary): from
    `frequencies` (radians per position, one for each pair) and `magnitude`, or from the options
    of rotary_frequencies()."""

    def __init__(self, rotary_dim, interleaved=False, frequencies=None, magnitude=1.0, **options):
        if frequencies is None:
            if magnitude != 1.0:
                options["magnitude"] = magnitude
            frequencies, magnitude = rotary_frequencies(rotary_dim, **options)
        elif options:
            raise ValueError("either frequencies or options to make them from")
        frequencies = [float(f) for f in frequencies]
        if len(frequencies) != rotary_dim // 2:
            raise ValueError("one frequency per pair")
        self.h = C.c_void_p()
        self.rotary_dim = rotary_dim
        check(lib().kvt_rotary_create(rotary_dim, 1 if interleaved else 0,
                                      (C.c_double * len(frequencies))(*frequencies), magnitude, C.byref(self.h)))

    def apply(self, x, positions, out, stream=None):
        """out[t, h] = x[t, h] rotated to positions[t] (int64); out may be x. -> out"""
        shape = tuple(x.shape)
        n, heads, dim = shape
        code = _code(x, "x")
        x_ptr, x_t, x_h = _rows(x, "x", shape, code)
        out_ptr, out_t, out_h = _rows(out, "out", shape, code)
        pos_ptr, device = _index(positions, "positions", (n,), "int64"), x.get_device()
        if out.get_device() != device or positions.get_device() != device:
            _refuse_elsewhere(device, dict(out=out, positions=positions))
        rc = lib().kvt_rotary_apply(self.h, device, code, x_ptr, x_t, x_h, out_ptr, out_t, out_h, pos_ptr, n, heads, dim,
                                    stream)
        if rc:
            check(rc)
        return out

    def close(self):
        if self.h:
            lib().kvt_rotary_destroy(self.h)
            self.h = C.c_void_p()

    __del__ = _quiet_close


def kv_append(cache, layer, layout, k, v, slots, rotary=None, positions=None, q=None, q_out=None, k_scale=1.0,
              v_scale=1.0, stream=None):
    """Writes the keys k (rotated to `positions`) and values v, [tokens, kv_heads, head_dim], to the
    rows slots[t] (int64: block * tokens_per_block + token; anything outside the cache: no row) of
    `layer` of a registered Cache, and the rotated queries q to q_out, in one launch
    (kvt_kv_append)."""
    n, dim = k.shape[0], layout.head_dim
    code = _code(k, "k")
    rows = (n, layout.n_kv_heads, dim)
    k_ptr, k_t, k_h = _rows(k, "k", rows, code)
    v_ptr, v_t, v_h = _rows(v, "v", rows, code)
    q_ptr = out_ptr = pos_ptr = None
    q_t = q_h = q_heads = out_t = out_h = 0
    if q is not None:
        if q_out is None:
            raise ValueError("q without q_out")
        q_heads = q.shape[1]
        q_ptr, q_t, q_h = _rows(q, "q", (n, q_heads, dim), code)
        out_ptr, out_t, out_h = _rows(q_out, "q_out", (n, q_heads, dim), code)
    if positions is not None:
        pos_ptr = _index(positions, "positions", (n,), "int64")
    slots_ptr, device = _index(slots, "slots", (n,), "int64"), cache.device
    if k.get_device() != device or v.get_device() != device or slots.get_device() != device or (
            q is not None and (q.get_device() != device or q_out.get_device() != device)) or (
            positions is not None and positions.get_device() != device):
        _refuse_elsewhere(device, dict(k=k, v=v, slots=slots, q=q, q_out=q_out, positions=positions))
    rc = lib().kvt_kv_append(cache.h, layer, layout.ref, rotary.h if rotary is not None else None, code, k_ptr, k_t, k_h,
                             v_ptr, v_t, v_h, q_ptr, q_t, q_h, q_heads, out_ptr, out_t, out_h, pos_ptr, slots_ptr, n,
                             k_scale, v_scale, stream)
    if rc:
        check(rc)


class DecodeAttention:
    """Attention of one new token per sequence over the paged cache (kvt_decode). One object serves
    all layers; every stream that launches it and every stream capture takes one of `workspaces`."""

    def __init__(self, device, layout, dtype, n_q_heads, max_seqs, softmax_scale=None, logit_cap=0.0, window=0,
                 workspaces=4):
        self.h = C.c_void_p()
        self.device, self.layout, self.n_q_heads, self.code = device, layout, n_q_heads, DTYPES[dtype]
        check(lib().kvt_decode_create(device, layout.ref, self.code, n_q_heads, softmax_scale or 0.0, logit_cap,
                                      window, max_seqs, workspaces, C.byref(self.h)))

    def run(self, cache, layer, q, block_tables, seq_lens, out, lse=None, max_len=0, k_scale=1.0, v_scale=1.0,
            stream=None):
        """q, out: [seqs, n_q_heads, head_dim]; block_tables: int32 [seqs, blocks]; seq_lens: int32 [seqs];
        lse: float32 [seqs, n_q_heads] or None. max_len: the longest length if known. -> out"""
        _code(q, "q")
        n, heads = q.shape[0], self.n_q_heads
        shape = (n, heads, self.layout.head_dim)
        columns = block_tables.shape[1] if block_tables.dim() == 2 else -1
        if columns < 0 or block_tables.shape[0] != n or block_tables.dtype != _types["int32"] or (
                columns > 1 and block_tables.stride(1) != 1):
            raise ValueError("block_tables: expected int32 [%d, blocks] with contiguous rows" % n)
        q_ptr, q_t, q_h = _rows(q, "q", shape, self.code)
        out_ptr, out_t, out_h = _rows(out, "out", shape, self.code)
        lens_ptr, lse_ptr = _index(seq_lens, "seq_lens", (n,), "int32"), None
        if lse is not None:
            lse_ptr = _index(lse, "lse", (n, heads), 2)
        device = self.device
        if q.get_device() != device or block_tables.get_device() != device or seq_lens.get_device() != device or (
                out.get_device() != device) or (lse is not None and lse.get_device() != device):
            _refuse_elsewhere(device, dict(q=q, block_tables=block_tables, seq_lens=seq_lens, out=out, lse=lse))
        rc = lib().kvt_decode_attention(
            self.h, cache.h, layer, q_ptr, q_t, q_h, block_tables.data_ptr(), block_tables.stride(0), columns, lens_ptr, n,
            max_len, k_scale, v_scale, out_ptr, out_t, out_h, lse_ptr, stream)
        if rc:
            check(rc)
        return out

    def release(self, stream=None):
        """Gives back the workspaces that `stream` and the captures made on it hold."""
        check(lib().kvt_decode_release(self.h, stream))

    def close(self):
        if self.h:
            lib().kvt_decode_destroy(self.h)
            self.h = C.c_void_p()

    __del__ = _quiet_close
