"""The operators on the registered cache (include/kvt_hip.h, "operators on the registered cache"):
rotary positions, the append of a step's keys and values to its pages, and the attention of one new
token over them.

Tensors are torch tensors on the cache's device (any strides; the elements of a row next to each
other), `stream` a hipStream_t handle as everywhere in this package (None: the default stream).
Sizes and types are checked here, everything else by the library."""
import ctypes as C

from . import binding
from .binding import KvLayoutStruct, RotaryOpts, _quiet_close, check, lib

DTYPES = {"bf16": 0, "f16": 1, "f32": 2, "e4m3": 3}
_TORCH_NAMES = {"torch.bfloat16": 0, "torch.float16": 1, "torch.float32": 2, "torch.float8_e4m3fn": 3}
_codes = {}          # torch dtype -> code, filled as they come
SCALINGS = {"plain": 0, "linear": 1, "bands": 2, "ramp": 3}


def _code(tensor, name):
    code = _codes.get(tensor.dtype)
    if code is None:
        code = _codes[tensor.dtype] = _TORCH_NAMES.get(str(tensor.dtype), -1)
    if code < 0:
        raise ValueError("%s: unsupported type %s" % (name, tensor.dtype))
    return code


def _rows(tensor, name, n_tokens, n_heads, dim, code):
    """(pointer, token stride, head stride) in bytes of a [tokens, heads, dim] tensor."""
    if tuple(tensor.shape) != (n_tokens, n_heads, dim) or _code(tensor, name) != code:
        raise ValueError("%s: got %s of %s, expected %s" % (name, tuple(tensor.shape), tensor.dtype,
                                                            (n_tokens, n_heads, dim)))
    t, h, e = tensor.stride()
    if e != 1 and dim > 1:
        raise ValueError("%s: the elements of a row must lie next to each other" % name)
    size = tensor.element_size()
    return tensor.data_ptr(), t * size, h * size


def _index(tensor, name, shape, dtype):
    """Pointer of a contiguous tensor of one type."""
    if tuple(tensor.shape) != shape or str(tensor.dtype) != dtype or not tensor.is_contiguous():
        raise ValueError("%s: expected a contiguous %s tensor of shape %s" % (name, dtype, shape))
    return tensor.data_ptr()


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
        n, heads, dim = x.shape
        code = _code(x, "x")
        check(lib().kvt_rotary_apply(self.h, x.get_device(), code, *_rows(x, "x", n, heads, dim, code),
                                     *_rows(out, "out", n, heads, dim, code),
                                     _index(positions, "positions", (n,), "torch.int64"), n, heads, dim, stream))
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
    q_args, q_heads, out_args = (None, 0, 0), 0, (None, 0, 0)
    if q is not None:
        q_heads = q.shape[1]
        q_args, out_args = _rows(q, "q", n, q_heads, dim, code), _rows(q_out, "q_out", n, q_heads, dim, code)
    check(lib().kvt_kv_append(cache.h, layer, layout.ref, rotary.h if rotary is not None else None, code,
                              *_rows(k, "k", n, layout.n_kv_heads, dim, code),
                              *_rows(v, "v", n, layout.n_kv_heads, dim, code), *q_args, q_heads, *out_args,
                              None if positions is None else _index(positions, "positions", (n,), "torch.int64"),
                              _index(slots, "slots", (n,), "torch.int64"), n, k_scale, v_scale, stream))


class DecodeAttention:
    """Attention of one new token per sequence over the paged cache (kvt_decode). One object serves
    all layers; every stream that launches it and every stream capture takes one of `workspaces`."""

    def __init__(self, device, layout, dtype, n_q_heads, max_seqs, softmax_scale=None, logit_cap=0.0, window=0,
                 workspaces=4):
        self.h = C.c_void_p()
        self.layout, self.n_q_heads, self.code = layout, n_q_heads, DTYPES[dtype]
        check(lib().kvt_decode_create(device, layout.ref, self.code, n_q_heads, softmax_scale or 0.0, logit_cap,
                                      window, max_seqs, workspaces, C.byref(self.h)))

    def run(self, cache, layer, q, block_tables, seq_lens, out, lse=None, max_len=0, k_scale=1.0, v_scale=1.0,
            stream=None):
        """q, out: [seqs, n_q_heads, head_dim]; block_tables: int32 [seqs, blocks]; seq_lens: int32 [seqs];
        lse: float32 [seqs, n_q_heads] or None. max_len: the longest length if known. -> out"""
        n, dim = q.shape[0], self.layout.head_dim
        if (block_tables.dim() != 2 or block_tables.shape[0] != n or str(block_tables.dtype) != "torch.int32"
                or (block_tables.shape[1] > 1 and block_tables.stride(1) != 1)):
            raise ValueError("block_tables: expected int32 [%d, blocks] with contiguous rows" % n)
        check(lib().kvt_decode_attention(
            self.h, cache.h, layer, *_rows(q, "q", n, self.n_q_heads, dim, self.code), block_tables.data_ptr(),
            block_tables.stride(0), block_tables.shape[1], _index(seq_lens, "seq_lens", (n,), "torch.int32"), n,
            max_len, k_scale, v_scale, *_rows(out, "out", n, self.n_q_heads, dim, self.code),
            None if lse is None else _index(lse, "lse", (n, self.n_q_heads), "torch.float32"), stream))
        return out

    def release(self, stream=None):
        """Gives back the workspaces that `stream` and the captures made on it hold."""
        check(lib().kvt_decode_release(self.h, stream))

    def close(self):
        if self.h:
            lib().kvt_decode_destroy(self.h)
            self.h = C.c_void_p()

    __del__ = _quiet_close
