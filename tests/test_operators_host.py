"""The host side of the operators on the paged cache: layouts of the cache shapes, frequencies of
rotary positions, and the calls that are refused before anything reaches a device. CPU only."""
import ctypes as C
import math

import numpy as np
import pytest

import kvt_amd
import operator_cases as oc
from kvt_amd import binding, ctypes_defs
from kvt_amd.ctypes_defs import ERR_INVALID, ERR_UNSUPPORTED


def _refused(code, fn, *args, **kw):
    with pytest.raises(kvt_amd.KvtError) as e:
        fn(*args, **kw)
    assert e.value.code == code, e.value
    return str(e.value)


def test_struct_sizes_match():
    assert kvt_amd.lib().kvt_abi_sizeof(7) == C.sizeof(binding.KvLayoutStruct)
    assert kvt_amd.lib().kvt_abi_sizeof(8) == C.sizeof(binding.RotaryOpts)


@pytest.mark.parametrize("dtype,size", [("bf16", 2), ("f16", 2), ("e4m3", 1)])
@pytest.mark.parametrize("layout", sorted(oc.SHAPES))
@pytest.mark.parametrize("n,block,heads,dim", [(7, 16, 8, 128), (3, 1, 1, 16), (5, 24, 3, 80), (1, 544, 2, 256)])
def test_layout_of_a_cache_shape_is_where_numpy_finds_the_rows(layout, dtype, size, n, block, heads, dim):
    a = np.arange(2 * n * block * heads * dim, dtype=np.int64).reshape(oc.cache_shape(layout, n, block, heads, dim))
    views = oc.kv_views(layout, a)
    s = kvt_amd.KvLayout(oc.SHAPES[layout], dtype, n, block, heads, dim).struct
    for which in (0, 1):
        for b, t, h in ((0, 0, 0), (n - 1, block - 1, heads - 1), (n // 2, block // 2, heads // 2)):
            at = b * s.block_stride + which * s.kv_stride + t * s.token_stride + h * s.head_stride
            assert at == int(views[which][b, t, h, 0]) * size


@pytest.mark.parametrize("shape", [ctypes_defs.SHAPE_DPSK_V32_SPARSE_MLA, ctypes_defs.SHAPE_KIMI_K3_MLA,
                                   ctypes_defs.SHAPE_TURBOQUANT, 0, 99])
def test_layouts_without_keys_and_values_per_head_are_refused(shape):
    _refused(ERR_UNSUPPORTED, kvt_amd.KvLayout, shape, "bf16", 8, 16, 1, 64)


@pytest.mark.parametrize("n,block,heads,dim", [(0, 16, 8, 128), (8, 0, 8, 128), (8, 16, 0, 128), (1 << 31, 16, 8, 128),
                                               (8, 65537, 8, 128), (8, 16, 65537, 128)])
def test_layout_sizes_out_of_range_are_refused(n, block, heads, dim):
    _refused(ERR_INVALID, kvt_amd.KvLayout, ctypes_defs.SHAPE_FLASH, "bf16", n, block, heads, dim)


@pytest.mark.parametrize("dim", [0, 8, 24, 100, 272])
def test_head_sizes_that_are_no_multiple_of_16_up_to_256_are_refused(dim):
    for shape in (ctypes_defs.SHAPE_FLASH, ctypes_defs.SHAPE_FLASHINFER):
        with pytest.raises(kvt_amd.KvtError) as e:
            kvt_amd.KvLayout(shape, "bf16", 8, 16, 8, dim)
        assert e.value.code in (ERR_INVALID, ERR_UNSUPPORTED)


def test_frequencies_are_the_formulas():
    d, base, f, length = 64, 10000.0, 8.0, 4096
    plain = [base ** (-2 * i / d) for i in range(d // 2)]
    got, m = kvt_amd.rotary_frequencies(d, base)
    assert np.allclose(got, plain, rtol=1e-14, atol=0) and m == 1.0
    got, m = kvt_amd.rotary_frequencies(d, base, "linear", f)
    assert np.allclose(got, [w / f for w in plain], rtol=1e-14, atol=0) and m == 1.0
    got, m = kvt_amd.rotary_frequencies(d, base, "bands", f, length)
    for w, g in zip(plain, got):
        turns = length * w / (2 * math.pi)
        mix = 0 if turns >= 4 else 1 if turns <= 1 else (4 - turns) / 3
        assert math.isclose(g, w * (1 - mix) + w / f * mix, rel_tol=1e-13)
    assert m == 1.0 and got[0] == plain[0] and math.isclose(got[-1], plain[-1] / f, rel_tol=1e-14)
    got, m = kvt_amd.rotary_frequencies(d, base, "ramp", f, length)
    pair = lambda turns: d * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = math.floor(pair(32)), math.ceil(pair(1))
    for i, (w, g) in enumerate(zip(plain, got)):
        mix = min(1, max(0, (i - lo) / (hi - lo)))
        assert math.isclose(g, w * (1 - mix) + w / f * mix, rel_tol=1e-13)
    assert math.isclose(m, 0.1 * math.log(f) + 1)
    assert kvt_amd.rotary_frequencies(d, base, "ramp", f, length, magnitude=0.5)[1] == 0.5
    assert kvt_amd.rotary_frequencies(d, base, "ramp", 0.5, length)[1] == 1.0


@pytest.mark.parametrize("dim,kw", [
    (0, {}), (3, {}), (258, {}), (64, dict(base=1.0)), (64, dict(base=math.nan)), (64, dict(scaling="linear", factor=0.0)),
    (64, dict(scaling="bands", factor=8.0)), (64, dict(scaling="ramp", factor=8.0, original_max_position=-1.0)),
    (64, dict(scaling="bands", factor=8.0, original_max_position=4096, low=4.0, high=4.0)),
    (64, dict(scaling="linear", factor=math.inf)), (64, dict(magnitude=-1.0))])
def test_frequencies_out_of_range_are_refused(dim, kw):
    _refused(ERR_INVALID, kvt_amd.rotary_frequencies, dim, **kw)


def test_rotations_out_of_range_are_refused():
    for bad in ([math.nan] + [1.0] * 31, [math.inf] + [1.0] * 31):
        _refused(ERR_INVALID, kvt_amd.Rotary, 64, frequencies=bad)
    _refused(ERR_INVALID, kvt_amd.Rotary, 64, frequencies=[1.0] * 32, magnitude=math.inf)
    with pytest.raises(ValueError):
        kvt_amd.Rotary(64, frequencies=[1.0] * 31)
    lib = kvt_amd.lib()
    assert lib.kvt_rotary_create(64, 0, None, 1.0, None) == ERR_INVALID
    lib.kvt_rotary_destroy(None)


@pytest.mark.parametrize("magnitude", [3.5e38, -1e39, 1e300])
def test_a_magnitude_beyond_32_bits_is_refused(magnitude):
    _refused(ERR_INVALID, kvt_amd.Rotary, 64, frequencies=[1.0] * 32, magnitude=magnitude)


# The calls below are refused on the host: the pointers are never followed.
P, POS = 1 << 20, 1 << 30


def _apply(r, **kw):
    a = dict(device=0, dtype=0, x=P, x_tok=1024, x_head=128, out=2 * P, out_tok=1024, out_head=128, positions=POS,
             n=64, heads=8, dim=64)
    a.update(kw)
    return kvt_amd.lib().kvt_rotary_apply(r.h if r else None, *a.values(), None)


def test_rotary_apply_refuses_on_the_host():
    r = kvt_amd.Rotary(64)
    assert _apply(None) == ERR_INVALID
    assert _apply(r, dtype=3) == ERR_UNSUPPORTED and _apply(r, dtype=9) == ERR_UNSUPPORTED
    assert _apply(r, dim=62) == ERR_INVALID and _apply(r, dim=257) == ERR_INVALID
    assert _apply(r, x=None) == ERR_INVALID and _apply(r, out=None) == ERR_INVALID
    assert _apply(r, positions=None) == ERR_INVALID and _apply(r, positions=POS + 4) == ERR_INVALID
    assert _apply(r, x=P + 1) == ERR_INVALID and _apply(r, out_tok=1025) == ERR_INVALID
    assert _apply(r, out_head=126) == ERR_INVALID                    # rows of the output meet
    assert _apply(r, out_tok=512) == ERR_INVALID
    assert _apply(r, out=P + 2) == ERR_INVALID                       # shares bytes with x
    assert _apply(r, out=P + 1024) == ERR_INVALID
    assert _apply(r, out=P, out_tok=2048) == ERR_INVALID             # in place with other strides
    assert _apply(r, n=1 << 62, x_tok=0, out_tok=1 << 20) == ERR_INVALID
    last = kvt_amd.lib().kvt_last_error()
    assert b"kvt_rotary_apply" in last


@pytest.mark.skipif(kvt_amd.device_count() > 0, reason="this check is for machines without a GPU")
def test_calls_that_are_right_need_a_device():
    r = kvt_amd.Rotary(64)
    assert _apply(r) == ctypes_defs.ERR_NO_DEVICE
    assert _apply(r, out=P) == ctypes_defs.ERR_NO_DEVICE             # in place
    # two halves of one wider tensor: interleaved, no byte shared
    assert _apply(r, x_tok=2048, out=P + 1024, out_tok=2048) == ctypes_defs.ERR_NO_DEVICE
    assert _apply(r, x=P + 1024, x_tok=2048, out=P, out_tok=2048) == ctypes_defs.ERR_NO_DEVICE


@pytest.mark.skipif(kvt_amd.device_count() > 0, reason="this check is for machines without a GPU")
def test_rows_of_one_wider_tensor_that_share_no_byte_are_told_apart():
    r, free = kvt_amd.Rotary(64), ctypes_defs.ERR_NO_DEVICE
    heads = dict(x_tok=2048, x_head=256, out_tok=2048, out_head=256)     # [tokens, 8, 2, 64]: x = w[:, :, 0]
    for off in (128, -128, 128 + 3 * 256, 2048 - 128, 128 - 5 * 2048, 70 * 2048 - 128):
        assert _apply(r, out=P + off, **heads) == free, off
    for off in (126, 2, -2, 256, -256, 130, 2048, -63 * 2048, 63 * 2048 + 7 * 256 + 126):
        assert _apply(r, out=P + off, **heads) == ERR_INVALID, off
    assert _apply(r, out=P + 63 * 2048 + 7 * 256 + 128, **heads) == free
    # heads in front of tokens, [8, 2, 64, 64]: x = w[:, 0]
    heads = dict(x_tok=128, x_head=16384, out_tok=128, out_head=16384)
    assert _apply(r, out=P + 8192, **heads) == free and _apply(r, out=P - 8192, **heads) == free
    for off in (8192 - 128, 8192 + 128, 8190, -8194, 128, 16384):
        assert _apply(r, out=P + off, **heads) == ERR_INVALID, off
    # interleaved at other strides: not worked out
    assert _apply(r, out=P + 128, x_tok=2048, x_head=256, out_tok=4096, out_head=256) == ERR_INVALID
    # strides of one token or of one head are none
    assert _apply(r, out=P, n=1, out_tok=4096) == free and _apply(r, out=P + 128, n=1, x_head=256, out_head=256) == free
    assert _apply(r, out=P, heads=1, x_head=2, out_head=6, x_tok=256, out_tok=256) == free
    assert _apply(r, out=P + 64, n=1, out_tok=4096) == ERR_INVALID
    assert _apply(r, out=P + 64, heads=1, x_head=2, x_tok=256, out_tok=256) == ERR_INVALID


@pytest.mark.skipif(kvt_amd.device_count() > 0, reason="this check is for machines without a GPU")
def test_rows_at_the_same_strides_are_refused_exactly_where_they_share_bytes():
    r, rng, seen = kvt_amd.Rotary(2), np.random.default_rng(31), set()
    for _ in range(4000):
        n, heads = (int(x) for x in rng.integers(1, 6, 2))
        strides = sorted(int(x) * 2 for x in rng.integers(2, 24, 2))
        tok, head = (strides if rng.random() < 0.5 else strides[::-1])
        off = 2 * int(rng.integers(-80, 80))
        rows = np.array([t * tok + h * head for t in range(n) for h in range(heads)])
        if np.diff(np.sort(rows)).min(initial=4) < 4:
            continue                                         # rows of the output itself meet
        got = _apply(r, x=P, x_tok=tok, x_head=head, out=P + off, out_tok=tok, out_head=head, n=n, heads=heads, dim=2)
        meet = (np.abs(rows[:, None] - (rows + off)[None]) < 4).any() and off != 0
        refusals = ERR_INVALID if meet else ctypes_defs.ERR_NO_DEVICE
        assert got == refusals or "overlap" in kvt_amd.lib().kvt_last_error().decode(), (n, heads, tok, head, off, got)
        seen.add((got, bool(meet)))
    assert (ERR_INVALID, True) in seen and (ctypes_defs.ERR_NO_DEVICE, False) in seen


def _append(layout, rotary, **kw):
    a = dict(dtype=0, k=P, k_tok=4096, k_head=256, v=P + 2048, v_tok=4096, v_head=256, q=4 * P, q_tok=8192, q_head=256,
             q_heads=32, q_out=8 * P, qo_tok=8192, qo_head=256, positions=POS, slots=2 * POS, n=8, k_scale=1.0,
             v_scale=1.0)
    a.update(kw)
    return kvt_amd.lib().kvt_kv_append(None, 0, layout.ref if layout else None, rotary.h if rotary else None,
                                       *a.values(), None)


def test_append_refuses_on_the_host():
    lay = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "bf16", 64, 16, 8, 128)
    lay8 = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "e4m3", 64, 16, 8, 128)
    r = kvt_amd.Rotary(128)
    said = lambda: kvt_amd.lib().kvt_last_error()  # noqa: E731
    assert _append(lay, r) == ERR_INVALID and b"null cache" in said()    # everything else is right
    assert _append(lay, None, q=None, q_heads=0, positions=None) == ERR_INVALID and b"null cache" in said()
    assert _append(lay8, r, k_scale=0.5) == ERR_INVALID and b"null cache" in said()
    assert _append(None, r) == ERR_INVALID and b"null layout" in said()
    assert _append(lay, r, dtype=2) == ERR_UNSUPPORTED and _append(lay, r, dtype=1) == ERR_UNSUPPORTED
    assert _append(lay, r, k_scale=2.0) == ERR_INVALID and b"scales" in said()
    for bad in (0.0, -1.0, math.nan, math.inf, 1e-39):
        assert _append(lay8, r, v_scale=bad) == ERR_INVALID and b"scales" in said()
    assert _append(lay, None) == ERR_INVALID and b"rotation" in said()
    assert _append(lay, kvt_amd.Rotary(256)) == ERR_INVALID and b"longer" in said()
    assert _append(lay, r, slots=None) == ERR_INVALID and b"slots" in said()
    assert _append(lay, r, positions=POS + 1) == ERR_INVALID and b"positions" in said()
    assert _append(lay, r, k=None) == ERR_INVALID and _append(lay, r, q_out=None) == ERR_INVALID
    assert _append(lay, r, q_out=P) == ERR_INVALID and b"shares bytes" in said()
    assert _append(lay, r, q_out=4 * P, qo_tok=16384) == ERR_INVALID and b"shares bytes" in said()
    # q rotated in place inside the fused tensor that holds k and v as well
    fused = dict(q=P, q_tok=12288, q_out=P, qo_tok=12288, k=P + 8192, k_tok=12288, v=P + 10240, v_tok=12288)
    assert _append(lay, r, **fused) == ERR_INVALID and b"null cache" in said()
    assert _append(lay, r, **dict(fused, k=P + 8000)) == ERR_INVALID and b"shares bytes with k" in said()


def test_index_arrays_inside_what_is_written_are_refused():
    lay, r = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "bf16", 64, 16, 8, 128), kvt_amd.Rotary(128)
    said = lambda: kvt_amd.lib().kvt_last_error()  # noqa: E731
    last = 8 * P + 7 * 8192 + 31 * 256 + 256                 # behind the last row of q_out
    for at in (8 * P - 56, 8 * P, 8 * P + 4096, last - 8):
        assert _append(lay, r, slots=at) == ERR_INVALID and b"q_out shares bytes with slots" in said()
        assert _append(lay, r, positions=at) == ERR_INVALID and b"q_out shares bytes with positions" in said()
    for at in (8 * P - 64, last):
        assert _append(lay, r, slots=at, positions=at) == ERR_INVALID and b"null cache" in said()
    r = kvt_amd.Rotary(64)
    for at in (2 * P, 2 * P - 8 * 63, 2 * P + 63 * 1024 + 1016):
        assert _apply(r, positions=at) == ERR_INVALID and b"out shares bytes with positions" in said()


@pytest.mark.skipif(kvt_amd.device_count() > 0, reason="this check is for machines without a GPU")
def test_more_rows_than_a_launch_can_have_are_refused_as_such():
    """A grid has fewer than 2^32 lanes: 16777215 workgroups of 256."""
    said, lanes = (lambda: kvt_amd.lib().kvt_last_error()), 16777215 * 256
    r, far = kvt_amd.Rotary(64), dict(out=P, positions=1 << 50)
    most = lanes // (8 * 4)                                  # 8 heads of four times two 16-byte pieces
    assert _apply(r, n=most, **far) == ctypes_defs.ERR_NO_DEVICE
    assert _apply(r, n=most + 1, **far) == ERR_INVALID and b"too many rows" in said()
    most = lanes // (8 * 32)                                 # unaligned: of 32 pairs
    assert _apply(r, n=most, x=P + 2, **dict(far, out=P + 2)) == ctypes_defs.ERR_NO_DEVICE
    assert _apply(r, n=most + 1, x=P + 2, **dict(far, out=P + 2)) == ERR_INVALID and b"too many rows" in said()
    lay, r = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "bf16", 64, 16, 8, 128), kvt_amd.Rotary(128)
    fused = dict(q=P, q_tok=12288, q_out=P, qo_tok=12288, k=P + 8192, k_tok=12288, v=P + 10240, v_tok=12288,
                 positions=1 << 50, slots=1 << 51)
    most = lanes // ((32 + 8 + 8) * 8)
    assert _append(lay, r, n=most, **fused) == ERR_INVALID and b"null cache" in said()
    assert _append(lay, r, n=most + 1, **fused) == ERR_INVALID and b"too many rows" in said()


def test_append_takes_queries_rotated_in_place_in_a_projection_that_is_fused_head_by_head():
    lay, r = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "bf16", 64, 16, 8, 128), kvt_amd.Rotary(128)
    w = dict(q=P, q_tok=6144, q_head=768, q_heads=8, q_out=P, qo_tok=6144, qo_head=768, k=P + 256, k_tok=6144, k_head=768,
             v=P + 512, v_tok=6144, v_head=768)                          # [tokens, 8, 3, 128]
    said = lambda: kvt_amd.lib().kvt_last_error()  # noqa: E731
    assert _append(lay, r, **w) == ERR_INVALID and b"null cache" in said()
    assert _append(lay, r, **dict(w, n=1)) == ERR_INVALID and b"null cache" in said()
    assert _append(lay, r, **dict(w, k=P + 254)) == ERR_INVALID and b"shares bytes with k" in said()
    assert _append(lay, r, **dict(w, v=P + 768)) == ERR_INVALID and b"shares bytes with v" in said()


@pytest.mark.parametrize("strides", [(0, 1 << 16, 256, 4096), (65536, 256, 256, 4096), (65536, 1 << 22, 255, 4096),
                                     (65536, 1 << 22, 4096, 128), (1 << 62, 1 << 61, 256, 4096)])
def test_layouts_whose_rows_meet_are_refused(strides):
    lay = kvt_amd.KvLayout(None, "bf16", 64, 16, 8, 128, strides=strides)
    assert _append(lay, kvt_amd.Rotary(128)) == ERR_INVALID
    assert b"null cache" not in kvt_amd.lib().kvt_last_error()


def test_decode_create_refuses_on_the_host():
    lay = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "bf16", 64, 16, 8, 128)
    lay8 = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "e4m3", 64, 16, 8, 128)
    new = kvt_amd.DecodeAttention
    _refused(ERR_UNSUPPORTED, new, 0, lay, "f16", 32, 4)             # not the cache's type
    _refused(ERR_UNSUPPORTED, new, 0, lay8, "f32", 32, 4)
    _refused(ERR_UNSUPPORTED, new, 0, lay8, "e4m3", 32, 4)
    for heads in (0, 7, 12, 8 * 65536):
        _refused(ERR_INVALID, new, 0, lay, "bf16", heads, 4)
    for kw in (dict(max_seqs=0), dict(max_seqs=65536), dict(workspaces=0), dict(workspaces=1025),
               dict(logit_cap=-1.0), dict(logit_cap=math.inf), dict(softmax_scale=math.nan), dict(softmax_scale=math.inf)):
        _refused(ERR_INVALID, new, 0, lay, "bf16", 32, **dict(dict(max_seqs=4), **kw))
    bad = kvt_amd.KvLayout(None, "bf16", 64, 16, 8, 128, strides=(65536, 1 << 22, 255, 4096))
    _refused(ERR_INVALID, new, 0, bad, "bf16", 32, 4)
    lib = kvt_amd.lib()
    assert lib.kvt_decode_create(0, lay.ref, 0, 32, 0.0, 0.0, 0, 4, 1, None) == ERR_INVALID
    assert lib.kvt_decode_create(0, None, 0, 32, 0.0, 0.0, 0, 4, 1, C.byref(C.c_void_p())) == ERR_INVALID
    assert lib.kvt_decode_attention(None, None, 0, P, 0, 0, P, 0, 1, P, 1, 0, 1.0, 1.0, P, 0, 0, None, None) == ERR_INVALID
    assert lib.kvt_decode_release(None, None) == ERR_INVALID
    lib.kvt_decode_destroy(None)


@pytest.mark.parametrize("kw", [dict(logit_cap=3e38), dict(softmax_scale=3e38), dict(softmax_scale=-3e38),
                                dict(softmax_scale=1.0, logit_cap=1e-39), dict(softmax_scale=1e30, logit_cap=1e-20)])
def test_scales_and_caps_whose_products_leave_32_bits_are_refused(kw):
    lay = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "bf16", 64, 16, 8, 128)
    _refused(ERR_INVALID, kvt_amd.DecodeAttention, 0, lay, "bf16", 32, 4, **kw)


@pytest.mark.skipif(kvt_amd.device_count() > 0, reason="this check is for machines without a GPU")
def test_decode_create_needs_a_device():
    lay = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "bf16", 64, 16, 8, 128)
    _refused(ctypes_defs.ERR_NO_DEVICE, kvt_amd.DecodeAttention, 0, lay, "bf16", 32, 4)


def test_the_binding_checks_sizes_and_types_before_the_library():
    import torch
    lay = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "bf16", 64, 16, 2, 64)
    r = kvt_amd.Rotary(64)
    rows, slots = torch.zeros((3, 2, 64), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)

    class NoCache:
        h = None

    ok = dict(k=rows, v=rows, slots=slots)
    for bad in (dict(v=rows[:2]), dict(v=rows.half()), dict(slots=slots.int()), dict(slots=slots[:2]),
                dict(k=rows.double()), dict(v=rows[..., ::2]), dict(k=rows[..., :32], v=rows[..., :32]),
                dict(q=rows), dict(q=rows, q_out=rows.float()), dict(rotary=r, positions=slots.float())):
        with pytest.raises(ValueError):
            kvt_amd.kv_append(NoCache, 0, lay, **dict(ok, **bad))
    with pytest.raises(ValueError):
        r.apply(rows, slots, rows[:2])
    with pytest.raises(ValueError):
        r.apply(rows, slots[:1], rows)
    with pytest.raises(ValueError):
        r.apply(rows.transpose(1, 2), slots, rows.transpose(1, 2))


def test_a_first_call_beside_another_threads_first_call(monkeypatch):
    """The table of torch types is there whole or not at all, wherever the thread that makes it is held back."""
    import threading

    import torch
    from kvt_amd import operators
    held, go_on, done = threading.Event(), threading.Event(), threading.Event()

    class Halting(dict):
        def update(self, *args, **kw):
            super().update(*args, **kw)
            held.set()
            go_on.wait(10)

    monkeypatch.setattr(operators, "_types", Halting())
    rows, slots = torch.zeros((3, 2, 64), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)

    def first():
        operators._code(rows, "k")
        held.set()
        done.set()

    thread = threading.Thread(target=first)
    thread.start()
    try:
        assert held.wait(10)
        assert operators._code(rows, "k") == 0
        assert operators._rows(rows, "k", (3, 2, 64), 0)[1:] == (256, 128)
        assert operators._index(slots, "slots", (3,), "int64") == slots.data_ptr()
    finally:
        go_on.set()
        thread.join()
    assert done.is_set()


class _On:
    """A tensor that says it is on some device."""

    def __init__(self, tensor, device):
        self._tensor, self._device = tensor, device

    def get_device(self):
        return self._device

    def __getattr__(self, name):
        return getattr(self._tensor, name)


def test_tensors_of_another_device_are_refused_by_the_binding():
    import torch
    lay, r = kvt_amd.KvLayout(ctypes_defs.SHAPE_FLASH, "bf16", 64, 16, 2, 64), kvt_amd.Rotary(64)

    class NoCache:
        h, device = None, 3

    rows = {n: torch.zeros((3, 2, 64), dtype=torch.bfloat16) for n in ("k", "v", "q", "q_out", "out")}
    rows.update((n, torch.zeros(3, dtype=torch.int64)) for n in ("slots", "positions"))
    rows.update(seq_lens=torch.zeros(3, dtype=torch.int32), block_tables=torch.zeros((3, 4), dtype=torch.int32),
                lse=torch.zeros((3, 2)))
    attention = object.__new__(kvt_amd.DecodeAttention)
    attention.h, attention.layout, attention.n_q_heads, attention.code, attention.device = C.c_void_p(), lay, 2, 0, 3
    calls = [(("k", "v", "slots", "positions", "q", "q_out"), lambda kw: kvt_amd.kv_append(NoCache, 0, lay, rotary=r, **kw)),
             (("q", "block_tables", "seq_lens", "out", "lse"), lambda kw: attention.run(NoCache, 0, **kw)),
             (("q", "positions", "out"), lambda kw: r.apply(kw["q"], kw["positions"], kw["out"]))]
    for names, call in calls:
        here = {n: _On(rows[n], 3) for n in names}
        said = _refused(ERR_INVALID, call, here) if names[0] != "q" or len(names) > 3 else ""
        assert "device" not in said                          # all on one device: the library's own refusal (no cache)
        for odd in names:
            for where in (1, -1):
                said = _refused(ERR_INVALID, call, dict(here, **{odd: _On(rows[odd], where)}))
                assert "not on one device" in said, (odd, where, said)
