"""Rotary positions and the append to the paged cache (kvt_rotary_apply, kvt_kv_append) against
their formulas in 64 bits on the CPU: types, cache layouts, head sizes and parts, strides, odd
token counts, padding, and everything around the written rows byte for byte. Needs a real MI355X."""
import numpy as np
import pytest

import checkers
import kvt_amd
import operator_cases as oc
from kvt_amd.ctypes_defs import ERR_INVALID, ERR_OUT_OF_RANGE

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, kind, g):
    return torch.randn(shape, generator=g, device="cuda").to(oc.torch_type(kind))


def _rotary(dim, inter, base=10000.0, **kw):
    freq, mag = kvt_amd.rotary_frequencies(dim, base=base, **kw)
    return kvt_amd.Rotary(dim, interleaved=inter, frequencies=freq, magnitude=mag), freq, mag


def _hold(got, exact, tol):
    bad = np.abs(got - exact) > tol
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - exact) / np.maximum(tol, 1e-300)).max()))


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("n,heads,dim,part", [(1, 1, 64, 64), (1, 40, 128, 128), (3, 5, 80, 80), (517, 9, 128, 128),
                                              (64, 3, 256, 64), (33, 2, 96, 18), (7, 1, 17, 6), (1000, 1, 16, 16),
                                              (130, 4, 250, 250), (2, 300, 64, 32)])
def test_rotation_is_the_formula(kind, inter, n, heads, dim, part):
    g = _gen(n * 1000 + dim)
    r, freq, mag = _rotary(part, inter, scaling="ramp", factor=8.0, original_max_position=4096)
    wide = _normal((n, heads + 2, dim), kind, g)
    x = wide[:, 1:heads + 1]
    pos = torch.randint(-1000, 200000, (n,), generator=g, device="cuda")
    out = torch.full((n, heads, dim), 7.0, device="cuda", dtype=x.dtype)
    r.apply(x, pos, out)
    exact, scale = oc.rotated(oc.wide(x), pos.cpu().numpy(), freq, mag, part, inter)
    _hold(oc.wide(out), exact, oc.rotation_tolerance(exact, scale, kind))
    assert torch.equal(out[..., part:], x[..., part:])
    # in place, inside the wider tensor, whose other rows keep their bytes
    before = wide.clone()
    r.apply(x, pos, x)
    assert torch.equal(x, out)
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, -1], before[:, -1])


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_far_positions_keep_their_angle(kind):
    """Positions up to 2^40 of integers that 32 bits do not hold; the angle is formed in 64 bits:
    2^-53 of 2^40 radians in the product and in the frequency is 2^-12 at most, of which the test's
    own 64-bit form has as much. Frequencies of a power of two keep both products exact."""
    g = _gen(5)
    freq = [2.0 * np.pi * 2.0 ** -(i + 3) for i in range(16)]
    r = kvt_amd.Rotary(32, frequencies=freq)
    x = _normal((257, 3, 64), kind, g)
    pos = torch.randint(0, 1 << 40, (257,), generator=g, device="cuda")
    out = r.apply(x, pos, torch.empty_like(x))
    turn = (pos.cpu().numpy()[:, None] % (1 << (np.arange(16) + 3))) / 2.0 ** (np.arange(16) + 3)   # exact
    xs = oc.wide(x)
    exact, scale = oc.rotated(xs, pos.cpu().numpy() * 0, freq, 1.0, 32, False)
    c, s = np.cos(2 * np.pi * turn)[:, None], np.sin(2 * np.pi * turn)[:, None]
    exact[..., :16] = xs[..., :16] * c - xs[..., 16:32] * s
    exact[..., 16:32] = xs[..., :16] * s + xs[..., 16:32] * c
    # the turns are frequency / (2 pi) rounded to 64 bits: 2^-53 of 2^37 turns, times 2 pi, at most 2^-13
    _hold(oc.wide(out), exact, oc.rotation_tolerance(exact, scale, kind) + 2.0 ** -13 * scale)


@pytest.mark.parametrize("shift", [1, 3, 8])
@pytest.mark.parametrize("inter", [False, True])
def test_rows_that_are_not_16_byte_aligned(shift, inter):
    g = _gen(shift)
    r, freq, mag = _rotary(64, inter)
    n, heads, dim = 19, 3, 64
    flat = _normal((n * (heads * dim + 5) + shift,), "bf16", g)
    x = flat[shift:shift + n * (heads * dim + 5)].view(n, -1)[:, :heads * dim].unflatten(1, (heads, dim))
    store = torch.zeros((n, heads + 1, dim + 1), device="cuda", dtype=torch.bfloat16)
    out = store[:, 1:, 1:]
    pos = torch.arange(n, device="cuda") * 37
    r.apply(x, pos, out)
    exact, scale = oc.rotated(oc.wide(x), pos.cpu().numpy(), freq, mag, 64, inter)
    _hold(oc.wide(out), exact, oc.rotation_tolerance(exact, scale, "bf16"))
    assert not store[:, 0].any() and not store[:, :, 0].any()


def _append_case(kind, cache_kind, layout, n, heads, kv_heads, dim, part, block, inter=False, k_scale=1.0,
                 v_scale=1.0, fused=True, seed=0):
    g = _gen(seed + n)
    r, freq, mag = _rotary(part, inter, base=500000.0, scaling="linear", factor=2.0)
    n_blocks = n // block + 5
    shape = oc.cache_shape(layout, n_blocks, block, kv_heads, dim)
    bits = torch.randint(0, 256, (int(np.prod(shape)) * (1 if cache_kind == "e4m3" else 2),), generator=g,
                         device="cuda", dtype=torch.uint8)
    cache = bits.view(oc.torch_type(cache_kind)).view(shape)
    before = bits.clone()
    if fused:
        all_rows = _normal((n, heads + 2 * kv_heads, dim), kind, g)
        q, k, v = all_rows[:, :heads], all_rows[:, heads:heads + kv_heads], all_rows[:, heads + kv_heads:]
    else:
        q, k, v = (_normal((n, h, dim), kind, g) for h in (heads, kv_heads, kv_heads))
    slots = torch.randperm(n_blocks * block, generator=g, device="cuda")[:n].contiguous()
    none = torch.rand((n,), generator=g, device="cuda") < 0.2
    slots[none] = torch.tensor([-1, -(1 << 62), n_blocks * block, 1 << 62], device="cuda")[
        torch.arange(n, device="cuda")[none] % 4]
    pos = torch.randint(0, 100000, (n,), generator=g, device="cuda")
    q_out = torch.empty((n, heads, dim), device="cuda", dtype=q.dtype)
    handle = kvt_amd.Cache(0, [[cache]], [bits.numel()])
    lay = kvt_amd.KvLayout(oc.SHAPES[layout], cache_kind, n_blocks, block, kv_heads, dim)
    kvt_amd.kv_append(handle, 0, lay, k, v, slots, rotary=r, positions=pos, q=q, q_out=q_out, k_scale=k_scale,
                      v_scale=v_scale)
    # the rows that were written
    ps, ss = pos.cpu().numpy(), slots.cpu().numpy()
    live = (ss >= 0) & (ss < n_blocks * block)
    views = oc.kv_views(layout, cache)
    got = [oc.wide(x[torch.from_numpy(ss[live] // block).cuda(), torch.from_numpy(ss[live] % block).cuda()]
                   if cache_kind != "e4m3" else
                   x.view(torch.uint8)[torch.from_numpy(ss[live] // block).cuda(),
                                       torch.from_numpy(ss[live] % block).cuda()].view(torch.float8_e4m3fn))
           for x in views]
    ke, kscale = oc.rotated(oc.wide(k), ps, freq, mag, part, inter)
    ve = oc.wide(v)
    ke, kscale, ve = ke[live] / k_scale, kscale[live] / k_scale, ve[live] / v_scale
    if cache_kind == "e4m3":
        assert np.abs(ke).max() < 440 and np.abs(ve).max() < 440
    # the scale's reciprocal and the product with it: two more roundings
    extra = 0 if cache_kind != "e4m3" else 2 * 2.0 ** -24
    _hold(got[0], ke, oc.rotation_tolerance(ke, kscale, cache_kind) + extra * kscale)
    _hold(got[1], ve, oc.HALF_STEP[cache_kind][0] * np.abs(ve) * (1 + 2.0 ** -10) + oc.HALF_STEP[cache_kind][1])
    if cache_kind == kind:
        assert np.array_equal(got[1], ve)
    qe, qscale = oc.rotated(oc.wide(q), ps, freq, mag, part, inter)
    _hold(oc.wide(q_out), qe, oc.rotation_tolerance(qe, qscale, kind))
    # every other byte of the cache is what it was
    width = torch.uint8 if cache_kind == "e4m3" else torch.int16
    now, was = bits.view(width).view(shape).clone(), before.view(width).view(shape)
    for a, b in zip(oc.kv_views(layout, now), oc.kv_views(layout, was)):
        at = (torch.from_numpy(ss[live] // block).cuda(), torch.from_numpy(ss[live] % block).cuda())
        a[at] = b[at]
    assert torch.equal(now, was)


@pytest.mark.parametrize("layout", sorted(oc.SHAPES))
@pytest.mark.parametrize("kind,cache_kind", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
def test_append_writes_the_rotated_rows_and_nothing_else(layout, kind, cache_kind):
    scales = (0.25, 1.7) if cache_kind == "e4m3" else (1.0, 1.0)
    _append_case(kind, cache_kind, layout, 83, 8, 2, 128, 128, 16, k_scale=scales[0], v_scale=scales[1])
    _append_case(kind, cache_kind, layout, 301, 5, 5, 80, 48, 5, inter=True, fused=False)


@pytest.mark.parametrize("n,heads,kv_heads,dim,part,block", [
    (1, 32, 8, 128, 128, 16), (2, 1, 1, 16, 2, 1), (257, 16, 2, 256, 64, 64), (40, 12, 4, 64, 22, 24),
    (1500, 1, 1, 16, 16, 128), (6, 128, 1, 192, 192, 544), (700, 3, 1, 16, 6, 8)])
@pytest.mark.parametrize("inter", [False, True])
def test_append_sizes(n, heads, kv_heads, dim, part, block, inter):
    _append_case("bf16", "bf16", "flash", n, heads, kv_heads, dim, part, block, inter=inter, seed=3)
    _append_case("bf16", "e4m3", "hnd", n, heads, kv_heads, dim, part, block, inter=inter, seed=4)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("kind,dim,part", [("bf16", 128, 128), ("f32", 128, 32), ("f16", 80, 48)])
def test_long_inputs(kind, dim, part, inter):
    """More than is expected to be left in a cache, and tokens that no workgroup begins with."""
    g = _gen(11)
    r, freq, mag = _rotary(part, inter)
    n = (140 << 20) // (9 * dim * (4 if kind == "f32" else 2))
    x = _normal((n, 9, dim), kind, g)
    pos = torch.randint(0, 100000, (n,), generator=g, device="cuda")
    out = r.apply(x, pos, torch.empty_like(x))
    some = torch.cat((torch.arange(64, device="cuda"), torch.randint(0, n, (2000,), generator=g, device="cuda"),
                      torch.arange(n - 64, n, device="cuda")))
    exact, scale = oc.rotated(oc.wide(x[some]), pos[some].cpu().numpy(), freq, mag, part, inter)
    _hold(oc.wide(out[some]), exact, oc.rotation_tolerance(exact, scale, kind))
    # all of it, by the rows one at a time being what they are together
    half = torch.empty_like(x)
    for a in range(0, n, 4096):
        r.apply(x[a:a + 4096], pos[a:a + 4096], half[a:a + 4096])
    assert torch.equal(half, out)


def test_append_without_rotation_or_queries_copies():
    g = _gen(1)
    cache = torch.zeros((2, 9, 16, 4, 64), device="cuda", dtype=torch.bfloat16)
    handle = kvt_amd.Cache(0, [[torch.zeros_like(cache)], [cache]], [cache.numel() * 2])
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", 9, 16, 4, 64)
    k, v = _normal((20, 4, 64), "bf16", g), _normal((20, 4, 64), "bf16", g)
    slots = torch.randperm(9 * 16, generator=g, device="cuda")[:20].contiguous()
    kvt_amd.kv_append(handle, 1, lay, k, v, slots)
    assert torch.equal(cache[0].flatten(0, 1)[slots], k) and torch.equal(cache[1].flatten(0, 1)[slots], v)
    # a broadcast row: one token's rows for all
    kvt_amd.kv_append(handle, 1, lay, k[:1].expand(20, 4, 64), v[:, :1].expand(20, 4, 64), slots)
    assert torch.equal(cache[0].flatten(0, 1)[slots], k[:1].expand(20, 4, 64))
    assert torch.equal(cache[1].flatten(0, 1)[slots], v[:, :1].expand(20, 4, 64))
    assert not handle._keep[0][0].any()                 # the other layer


def test_append_saturates_and_keeps_nan_like_the_converting_pack():
    """All bf16 patterns as values: the cache's bytes are those of kvt_launch_copy_d2h_bf16_to_fp8."""
    pats = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    v = pats.view(256, 1, 256)
    cache = torch.zeros((256, 1, 2, 1, 256), device="cuda", dtype=torch.uint8)
    handle = kvt_amd.Cache(0, [[cache]], [cache.numel()])
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_RAGGED_FLASH, "e4m3", 256, 1, 1, 256)
    kvt_amd.kv_append(handle, 0, lay, v, v, torch.arange(256, device="cuda"))
    want = torch.empty(65536, device="cuda", dtype=torch.uint8)
    zero, n = torch.zeros(1, device="cuda", dtype=torch.int64), torch.tensor([65536], device="cuda")
    assert kvt_amd.lib().kvt_launch_copy_d2h_bf16_to_fp8(pats.data_ptr(), want.data_ptr(), zero.data_ptr(),
                                                         zero.data_ptr(), n.data_ptr(), 1, 0, 0, None) == 0
    torch.cuda.synchronize()
    assert torch.equal(cache[:, 0, 0, 0].flatten(), want) and torch.equal(cache[:, 0, 1, 0].flatten(), want)


@pytest.mark.parametrize("n", [1, 5, 300])
def test_a_projection_that_is_fused_head_by_head(n):
    """[tokens, heads, 3, dim] with its queries rotated in place beside keys and values."""
    g = _gen(21)
    w = _normal((n, 6, 3, 64), "bf16", g)
    before = w.clone()
    q, k, v = w[:, :, 0], w[:, :, 1], w[:, :, 2]
    r, pos = kvt_amd.Rotary(64), torch.randint(0, 9999, (n,), generator=g, device="cuda")
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", 30, 16, 6, 64)
    slots = torch.randperm(480, generator=g, device="cuda")[:n].contiguous()
    caches = [torch.zeros((2, 30, 16, 6, 64), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    handles = [kvt_amd.Cache(0, [[c]], [c.numel() * 2]) for c in caches]
    q_out = torch.empty((n, 6, 64), device="cuda", dtype=torch.bfloat16)
    kvt_amd.kv_append(handles[0], 0, lay, k.contiguous(), v.contiguous(), slots, rotary=r, positions=pos, q=q.contiguous(),
                      q_out=q_out)
    kvt_amd.kv_append(handles[1], 0, lay, k, v, slots, rotary=r, positions=pos, q=q, q_out=q)
    assert torch.equal(caches[0], caches[1]) and torch.equal(q, q_out) and torch.equal(w[:, :, 1:], before[:, :, 1:])
    # from one third of it to another
    r.apply(before[:, :, 0], pos, before[:, :, 2])
    assert torch.equal(before[:, :, 2], q_out) and torch.equal(before[:, :, 1], k)


def test_no_tokens_is_no_launch():
    cache = torch.zeros((2, 4, 16, 2, 64), device="cuda", dtype=torch.bfloat16)
    handle = kvt_amd.Cache(0, [[cache]], [cache.numel() * 2])
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", 4, 16, 2, 64)
    none = torch.zeros((0, 2, 64), device="cuda", dtype=torch.bfloat16)
    kvt_amd.kv_append(handle, 0, lay, none, none, torch.zeros(0, device="cuda", dtype=torch.int64))
    r = kvt_amd.Rotary(64)
    r.apply(none, torch.zeros(0, device="cuda", dtype=torch.int64), none.clone())
    torch.cuda.synchronize()
    assert not cache.any()


def test_append_refusals_that_need_a_cache():
    cache = torch.zeros((2, 4, 16, 2, 64), device="cuda", dtype=torch.bfloat16)
    handle = kvt_amd.Cache(0, [[cache]], [cache.numel() * 2])
    rows = torch.ones((3, 2, 64), device="cuda", dtype=torch.bfloat16)
    slots = torch.arange(3, device="cuda")
    big = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", 5, 16, 2, 64)
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", 4, 16, 2, 64)
    second = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", 4, 16, 2, 64, tensor=1)
    for layer, layout, code in ((0, big, ERR_OUT_OF_RANGE), (1, lay, ERR_OUT_OF_RANGE), (0, second, ERR_OUT_OF_RANGE)):
        with pytest.raises(kvt_amd.KvtError) as e:
            kvt_amd.kv_append(handle, layer, layout, rows, rows, slots)
        assert e.value.code == code
    odd = torch.zeros(cache.numel() + 8, device="cuda", dtype=torch.bfloat16)[1:]
    unaligned = kvt_amd.Cache(0, [[odd]], [cache.numel() * 2])
    with pytest.raises(kvt_amd.KvtError) as e:
        kvt_amd.kv_append(unaligned, 0, lay, rows, rows, slots)
    assert e.value.code == ERR_INVALID
    with pytest.raises(kvt_amd.KvtError) as e:           # plain host memory
        host = torch.ones((3, 2, 64), dtype=torch.bfloat16)
        kvt_amd.kv_append(handle, 0, lay, host, host, slots)
    assert e.value.code == ERR_INVALID
    inside = cache.flatten()[-3 * 2 * 64:].view(3, 2, 64)
    r, pos = kvt_amd.Rotary(64), torch.zeros(3, device="cuda", dtype=torch.int64)
    for rotated in (dict(k=inside, v=rows), dict(k=rows, v=inside),
                    dict(k=rows, v=rows, q=rows.clone(), q_out=inside, rotary=r, positions=pos),
                    dict(k=rows, v=rows, q=inside, q_out=rows.clone(), rotary=r, positions=pos)):
        with pytest.raises(kvt_amd.KvtError) as e:       # rows of the cache itself
            kvt_amd.kv_append(handle, 0, lay, slots=slots, **rotated)
        assert e.value.code == ERR_INVALID and "the cache's tensor" in str(e.value)
    with pytest.raises(ValueError):
        kvt_amd.kv_append(handle, 0, lay, rows, rows[:2], slots)
    with pytest.raises(ValueError):
        kvt_amd.kv_append(handle, 0, lay, rows, rows, slots.int())
    torch.cuda.synchronize()
    assert not cache.any()


def test_slots_and_positions_inside_the_cache_are_refused():
    cache = torch.zeros((2, 4, 16, 2, 64), device="cuda", dtype=torch.bfloat16)
    handle = kvt_amd.Cache(0, [[cache]], [cache.numel() * 2])
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", 4, 16, 2, 64)
    rows, slots = torch.ones((3, 2, 64), device="cuda", dtype=torch.bfloat16), torch.arange(3, device="cuda")
    inside = cache.view(torch.int64).flatten()[-3:]
    r = kvt_amd.Rotary(64)
    for kw in (dict(slots=inside), dict(slots=slots, rotary=r, positions=inside)):
        with pytest.raises(kvt_amd.KvtError) as e:
            kvt_amd.kv_append(handle, 0, lay, rows, rows, **kw)
        assert e.value.code == ERR_INVALID and "the cache's tensor shares bytes" in str(e.value)
    torch.cuda.synchronize()
    assert not cache.any()


def test_host_arrays_are_taken_where_the_device_can_read_them():
    cache = torch.zeros((2, 4, 16, 2, 64), device="cuda", dtype=torch.bfloat16)
    handle = kvt_amd.Cache(0, [[cache]], [cache.numel() * 2])
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", 4, 16, 2, 64)
    rows = _normal((3, 2, 64), "bf16", _gen(31))
    slots = torch.tensor([5, 40, 17])
    pinned, host = slots.pin_memory(), rows.cpu()
    kvt_amd.kv_append(handle, 0, lay, rows, rows, pinned)
    torch.cuda.synchronize()
    assert torch.equal(cache[0].flatten(0, 1)[slots.cuda()], rows)
    st, graph = checkers.side_stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):                 # also where the runtime is not asked
        for kw in (dict(slots=slots), dict(slots=pinned, k=host)):
            with pytest.raises(kvt_amd.KvtError) as e:
                kvt_amd.kv_append(handle, 0, lay, **dict(dict(k=rows, v=rows), **kw), stream=st.cuda_stream)
            assert e.value.code == ERR_INVALID
        kvt_amd.kv_append(handle, 0, lay, rows, rows, pinned, stream=st.cuda_stream)
    cache.zero_()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache[1].flatten(0, 1)[slots.cuda()], rows)


def test_captured_append_reads_its_arrays_anew_on_every_replay():
    st = checkers.side_stream()
    g = _gen(9)
    cache = torch.zeros((2, 40, 16, 2, 64), device="cuda", dtype=torch.float16)
    handle = kvt_amd.Cache(0, [[cache]], [cache.numel() * 2])
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "f16", 40, 16, 2, 64)
    r, _, _ = _rotary(64, False)
    q, k, v = (_normal((33, h, 64), "f16", g) for h in (6, 2, 2))
    slots, pos = torch.full((33,), -1, device="cuda"), torch.zeros(33, device="cuda", dtype=torch.int64)
    q_out = torch.empty_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        kvt_amd.kv_append(handle, 0, lay, k, v, slots, rotary=r, positions=pos, q=q, q_out=q_out,
                          stream=torch.cuda.current_stream().cuda_stream)
    for step in range(4):
        k.copy_(_normal(k.shape, "f16", g))
        pos.copy_(torch.randint(0, 9999, (33,), generator=g, device="cuda"))
        slots.copy_(torch.randperm(640, generator=g, device="cuda")[:33])
        graph.replay()
        torch.cuda.synchronize()
        again, q_again = cache.clone(), torch.empty_like(q)
        other = kvt_amd.Cache(0, [[again]], [cache.numel() * 2])
        kvt_amd.kv_append(other, 0, lay, k, v, slots, rotary=r, positions=pos, q=q, q_out=q_again)
        torch.cuda.synchronize()
        assert torch.equal(q_out, q_again) and torch.equal(cache, again)
        assert torch.equal(cache[1].flatten(0, 1)[slots], v)
