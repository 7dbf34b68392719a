"""Attention of one new token over the paged cache (kvt_decode_attention) against its formula in
64 bits on the CPU: types, layouts, head counts and sizes, lengths around every boundary, pages that
end inside a tile, windows, caps, rows that see nothing, rows that must not be looked at, splits,
streams and graphs. Needs a real MI355X."""
import concurrent.futures

import numpy as np
import pytest

import checkers
import kvt_amd
import operator_cases as oc
from kvt_amd.ctypes_defs import ERR_INVALID, ERR_OUT_OF_RANGE, ERR_UNSUPPORTED

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


class Case:
    """A cache in which every row that belongs to no sequence is NaN, and tables into it."""

    def __init__(self, kind, cache_kind, layout, lens, heads, kv_heads, dim, block, seed=0, spread=2.0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed * 7919 + dim + heads)
        self.kind, self.layout, self.block, self.lens = kind, layout, block, [int(n) for n in lens]
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        pages = [max(0, -(-n // block)) for n in self.lens]
        self.n_blocks = sum(pages) + 2
        shape = oc.cache_shape(layout, self.n_blocks, block, kv_heads, dim)
        self.cache_type = oc.torch_type(cache_kind)
        size = 1 if cache_kind == "e4m3" else 2
        width = torch.uint8 if size == 1 else torch.int16
        nan = {"bf16": 0x7FC0, "f16": 0x7E00, "e4m3": 0x7F}[cache_kind]
        self.cache = torch.full(shape, nan, device="cuda", dtype=width)
        perm = torch.randperm(self.n_blocks, generator=g, device="cuda").cpu().numpy()
        cols = max(pages + [1])
        self.tables = np.full((len(lens), cols), -1, dtype=np.int32)
        at = 0
        views = oc.kv_views(layout, self.cache)
        self.plain = [np.zeros((self.n_blocks, block, kv_heads, dim)) for _ in views]
        for b, n in enumerate(self.lens):
            ids = perm[at:at + pages[b]]
            at += pages[b]
            self.tables[b, :len(ids)] = ids
            if n <= 0:
                continue
            t = np.arange(n)
            where = (torch.from_numpy(ids[t // block]).cuda(), torch.from_numpy(t % block).cuda())
            for view, plain in zip(views, self.plain):
                rows = torch.randn((n, kv_heads, dim), generator=g, device="cuda").to(self.cache_type)
                view[where] = rows.view(width)
                plain[ids[t // block], t % block] = oc.wide(rows)
        self.q = (spread * torch.randn((len(lens), heads, dim), generator=g, device="cuda")).to(oc.torch_type(kind))
        self.d_tables = torch.from_numpy(self.tables).cuda()
        self.d_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.handle = kvt_amd.Cache(0, [[self.cache]], [self.cache.numel() * size])
        self.lay = kvt_amd.KvLayout(oc.SHAPES[layout], cache_kind, self.n_blocks, block, kv_heads, dim)

    def operator(self, **kw):
        kw.setdefault("max_seqs", len(self.lens))
        return kvt_amd.DecodeAttention(0, self.lay, self.kind, self.heads, **kw)

    def buffers(self):
        out = torch.full_like(self.q, 77.0)
        return out, torch.full((len(self.lens), self.heads), 77.0, device="cuda")

    def exact(self, **kw):
        scale = kw.pop("scale", None) or self.dim ** -0.5
        return oc.decode_exact(oc.wide(self.q), *self.plain, self.tables, self.lens, self.block, scale, **kw)

    def check(self, op, exact, max_len=0, **kw):
        out, lse = self.buffers()
        op.run(self.handle, 0, self.q, self.d_tables, self.d_lens, out, lse=lse, max_len=max_len, **kw)
        hold(out, lse, exact, self.kind)
        return out, lse


def hold(out, lse, exact, kind):
    eo, el, measure = exact
    to, tl = oc.decode_tolerance(eo, el, measure, kind)
    go, gl = oc.wide(out), oc.wide(lse)
    assert np.isfinite(go).all()
    off = np.abs(go - eo)
    assert (off <= to).all(), ("out", float(np.max(off / np.maximum(to, 1e-300))))
    none = np.isneginf(el)
    assert np.array_equal(np.isneginf(gl), none)
    off = np.abs(np.where(none, 0, gl) - np.where(none, 0, el))
    assert (off <= tl).all(), ("lse", float(np.max(off / np.maximum(tl, 1e-300))))


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 160, 255, 257, 300, 513, 700, -3]


@pytest.mark.parametrize("layout", sorted(oc.SHAPES))
@pytest.mark.parametrize("kind,cache_kind", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
def test_decode_is_the_formula(layout, kind, cache_kind):
    c = Case(kind, cache_kind, layout, LENS, 8, 2, 128, 16)
    scales = dict(k_scale=0.5, v_scale=1.7) if cache_kind == "e4m3" else {}
    exact = c.exact(**scales)
    op = c.operator()
    whole = c.check(op, exact, **scales)
    for max_len in (1, 128, 700, 100000):        # the caller's word changes nothing but the split
        c.check(op, exact, max_len=max_len, **scales)
    again = c.check(op, exact, **scales)
    assert torch.equal(whole[0], again[0]) and torch.equal(whole[1], again[1])


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (12, 4), (7, 1), (15, 3), (16, 1), (17, 1), (40, 2),
                                            (64, 2), (128, 1)])
@pytest.mark.parametrize("cache_kind", ["bf16", "e4m3"])
def test_head_counts(heads, kv_heads, cache_kind):
    c = Case("bf16", cache_kind, "flash", [0, 1, 77, 300, 33], heads, kv_heads, 64, 16, seed=1)
    c.check(c.operator(), c.exact())


@pytest.mark.parametrize("heads,kv_heads", [(16, 1), (32, 2), (20, 1), (48, 1), (66, 2), (100, 1)])
@pytest.mark.parametrize("kind,cache_kind,dim", [("bf16", "bf16", 256), ("f16", "e4m3", 256), ("f16", "f16", 144),
                                                 ("bf16", "bf16", 128)])
def test_many_heads_of_wide_rows(heads, kv_heads, kind, cache_kind, dim):
    c = Case(kind, cache_kind, "hnd", [1, 700, 0, 129], heads, kv_heads, dim, 16, seed=19)
    c.check(c.operator(), c.exact())


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 144, 160, 192, 224, 256])
@pytest.mark.parametrize("kind,cache_kind", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3")])
def test_head_sizes(dim, kind, cache_kind):
    c = Case(kind, cache_kind, "pages", [1, 40, 333, 0, 128], 6, 2, dim, 16, seed=2)
    c.check(c.operator(), c.exact())


@pytest.mark.parametrize("block", [1, 2, 3, 5, 7, 8, 16, 24, 32, 33, 64, 128, 544])
@pytest.mark.parametrize("layout", ["hnd", "ragged"])
def test_block_sizes(block, layout):
    c = Case("bf16", "bf16", layout, [1, 5, 31, 100, 129, 600, 1100], 4, 2, 64, block, seed=3)
    c.check(c.operator(), c.exact())


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 128, 500, 5000])
def test_windows(window):
    c = Case("bf16", "bf16", "flash", LENS + [1500], 8, 2, 64, 16, seed=4)
    op = c.operator(window=window)
    exact = c.exact(window=window)
    c.check(op, exact)
    c.check(op, exact, max_len=1500)
    # pages in front of the window may have been given back: their ids are not looked at
    for b, n in enumerate(c.lens):
        c.tables[b, :max(0, n - window) // c.block] = 1 << 30
    c.d_tables.copy_(torch.from_numpy(c.tables))
    c.check(op, exact)


@pytest.mark.parametrize("cap", [0.5, 30.0])
@pytest.mark.parametrize("scale", [0.02, 1.0, -0.3])
def test_cap_and_scale(cap, scale):
    c = Case("bf16", "bf16", "flash", [1, 40, 333, 0, 128], 8, 2, 64, 16, seed=5)
    exact = c.exact(scale=scale, cap=cap)
    c.check(c.operator(softmax_scale=scale, logit_cap=cap), exact)
    c.check(c.operator(softmax_scale=scale), c.exact(scale=scale))


def test_pages_outside_the_cache_are_not_seen():
    c = Case("bf16", "bf16", "hnd", [100, 64, 33, 700, 16], 4, 2, 64, 16, seed=6)
    c.tables[0, 1], c.tables[0, 6] = -1, c.n_blocks          # in the middle, and the last
    c.tables[1, :] = np.int32(-2 ** 31)                      # all of a sequence
    c.tables[3, ::2] = np.int32(2 ** 31 - 1)
    c.tables[4, 0] = c.n_blocks
    c.d_tables.copy_(torch.from_numpy(c.tables))
    exact = c.exact()
    assert np.isneginf(exact[1][1]).all() and np.isneginf(exact[1][4]).all()
    op = c.operator()
    for max_len in (0, 1):
        out, _ = c.check(op, exact, max_len=max_len)
        assert not out[1].any() and not out[4].any()


def test_lengths_beyond_the_table_end_with_it():
    c = Case("bf16", "bf16", "flash", [100, 64, 320], 4, 2, 64, 16, seed=7)
    c.tables = c.tables[:, :20].copy()
    for b, pages in enumerate((7, 4, 20)):                   # the columns behind a sequence's pages: its first page
        c.tables[b, pages:] = c.tables[b, 0]
    c.d_tables = torch.from_numpy(c.tables).cuda()
    for plain, view in zip(c.plain, oc.kv_views("flash", c.cache)):
        rows = torch.nan_to_num(view.view(torch.bfloat16))   # the first page of sequence 0 has no NaN to meet
        view.copy_(rows.view(torch.int16))
        plain[:] = oc.wide(rows)
    c.lens = [2 ** 31 - 1, 100000, 321]
    c.d_lens = torch.tensor(c.lens, dtype=torch.int32, device="cuda")
    c.check(c.operator(), c.exact())
    # no table at all: nothing is seen
    out, lse = c.buffers()
    c.operator().run(c.handle, 0, c.q, c.d_tables[:, :0].contiguous(), c.d_lens, out, lse=lse)
    assert not out.any() and torch.isneginf(lse).all()


def test_the_same_pages_in_several_sequences():
    c = Case("bf16", "bf16", "flash", [300, 300, 300, 10], 4, 2, 64, 16, seed=8)
    c.tables[1] = c.tables[0]
    c.tables[2, :] = c.tables[0, 0]                          # one page again and again
    c.lens[3] = 10
    c.d_tables.copy_(torch.from_numpy(c.tables))
    c.check(c.operator(), c.exact())


def test_strided_and_unaligned_queries_and_outputs():
    c = Case("bf16", "bf16", "flash", [1, 40, 333, 0, 128, 900], 8, 2, 80, 16, seed=9)
    exact, op = c.exact(), c.operator()
    n = len(c.lens)
    for shift, pad in ((0, 16), (1, 1), (4, 4), (8, 0)):
        store = torch.zeros((n, 3, 8, 80 + pad + shift), device="cuda", dtype=torch.bfloat16)
        q = store[:, 1, :, shift:shift + 80]
        q.copy_(c.q)
        c.q = q
        out_store = torch.full((n, 9, 80 + pad + shift), 5.0, device="cuda", dtype=torch.bfloat16)
        out = out_store[:, 1:, shift:shift + 80]
        lse = c.buffers()[1]
        op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, lse=lse)
        hold(out, lse, exact, "bf16")
        assert (out_store[:, 0] == 5).all() and (out_store[:, :, :shift] == 5).all()
        assert (out_store[:, :, shift + 80:] == 5).all()
    pad_tables = torch.full((n, c.tables.shape[1] + 13), -1, device="cuda", dtype=torch.int32)
    pad_tables[:, :c.tables.shape[1]] = c.d_tables
    c.d_tables = pad_tables[:, :c.tables.shape[1]]           # rows further apart than they are long
    c.check(op, exact)


@pytest.mark.parametrize("max_len", [0, 1])
@pytest.mark.parametrize("where", ["alone", "all", "a whole part", "beside minus infinity"])
def test_scores_that_are_nan_and_nothing_else(where, max_len):
    c = Case("bf16", "bf16", "flash", [1 if where == "alone" else 700, 33], 4, 1, 64, 16, seed=23)
    k = oc.kv_views("flash", c.cache)[0].view(torch.bfloat16)
    n = c.lens[0]
    at = {"alone": range(n), "all": range(n), "a whole part": range(512, 640), "beside minus infinity": range(n)}[where]
    c.q[0] = c.q[0].abs() + 0.5
    for t in at:
        k[int(c.tables[0, t // 16]), t % 16][0, 3] = float("-inf" if where.startswith("beside") and t != 300 else "nan")
    out, lse = c.buffers()
    c.operator().run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, lse=lse, max_len=max_len)
    assert np.isnan(oc.wide(out)[0]).all() and np.isnan(oc.wide(lse)[0]).all()
    exact = oc.decode_exact(oc.wide(c.q)[1:], *c.plain, c.tables[1:], [33], 16, 64 ** -0.5)
    hold(out[1:], lse[1:], exact, "bf16")


def test_infinities_and_nan_that_are_seen_follow_the_formula():
    c = Case("bf16", "bf16", "flash", [200, 200, 200, 200], 4, 1, 64, 16, seed=10)
    k, v = (x.view(torch.bfloat16) for x in oc.kv_views("flash", c.cache))

    def at(b, t):
        return int(c.tables[b, t // 16]), t % 16

    k[at(0, 150)][0, 3] = float("nan")                       # a NaN score: all of the row
    c.q[1] = c.q[1].abs() + 0.5
    k[at(1, 3)][0, 5] = float("-inf")                        # a score of minus infinity: weight zero
    v[at(2, 60)][0, 7] = float("inf")                        # one dim of V
    c.q[3] = c.q[3].abs() + 0.5
    for t in range(200):
        k[at(3, t)][0, 0] = float("-inf")                    # every score minus infinity
    for max_len in (0, 1):
        out, lse = c.buffers()
        c.operator().run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, lse=lse, max_len=max_len)
        o, l = oc.wide(out), oc.wide(lse)
        assert np.isnan(o[0]).all() and np.isnan(l[0]).all()
        assert np.isfinite(o[1]).all() and np.isfinite(l[1]).all()
        assert np.isposinf(o[2][:, 7]).all() and np.isfinite(np.delete(o[2], 7, axis=1)).all()
        assert np.isnan(o[3]).all() and np.isneginf(l[3]).all()
    plain = [p.copy() for p in c.plain]
    b, r = at(1, 3)
    plain[0][b, r, 0, 5] = -1e30
    exact = oc.decode_exact(oc.wide(c.q)[1:2], *plain, c.tables[1:2], [200], 16, 64 ** -0.5)
    hold(out[1:2], lse[1:2], exact, "bf16")


@pytest.mark.parametrize("kind,cache_kind,value", [("bf16", "bf16", "inf"), ("f16", "f16", "-inf"), ("bf16", "bf16", "nan"),
                                                   ("bf16", "e4m3", "nan"), ("f16", "e4m3", "nan")])
@pytest.mark.parametrize("at,high", [(5, 6), (5, 40), (40, 5), (5, 133), (133, 5), (5, 590), (590, 5), (300, 301)])
def test_infinities_and_nan_in_v_come_through_wherever_a_sequence_is_split(kind, cache_kind, value, at, high):
    """One token's weight leaves nothing of the others' in 32 bits (their scores are 2000 below), in the same tile, in
    another wavefront's, in a later tile, in another workgroup's share: what is not finite in another's V shows."""
    c = Case(kind, cache_kind, "flash", [600, 77], 4, 1, 64, 16, seed=26)
    k, v = (x.view(c.cache_type) for x in oc.kv_views("flash", c.cache))
    page = lambda t: (int(c.tables[0, t // 16]), t % 16)  # noqa: E731
    c.q[0, :, 0] = 80.0
    k[page(high)][0, 0] = 200.0
    v[page(at)][0, 7] = float(value)
    row = oc.wide(v[page(high)])[0]
    rest = oc.decode_exact(oc.wide(c.q)[1:], *c.plain, c.tables[1:], [77], 16, 64 ** -0.5)
    for max_len in (0, 1):
        out, lse = c.buffers()
        c.operator().run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, lse=lse, max_len=max_len)
        got = oc.wide(out)[0]
        assert np.array_equal(got[:, 7], np.full(4, float(value)), equal_nan=True), (max_len, got[:, 7])
        # the others: the row of the one token that counts, its sums rounded a few times in 32 bits
        got, want = np.delete(got, 7, axis=1), np.delete(row, 7)
        rel, floor = oc.HALF_STEP[kind]
        assert (np.abs(got - want) <= rel * np.abs(want) + floor + 2.0 ** -15 * np.abs(want)).all()
        hold(out[1:], lse[1:], rest, kind)


@pytest.mark.parametrize("at", [3, 9000, 20010])
def test_infinities_in_v_come_through_the_join_in_two_steps(at):
    c = Case("bf16", "bf16", "flash", [20011], 64, 1, 128, 16, seed=27)
    k, v = (x.view(torch.bfloat16) for x in oc.kv_views("flash", c.cache))
    c.q[0, :, 0] = 80.0
    k[int(c.tables[0, 10001 // 16]), 10001 % 16][0, 0] = 300.0
    v[int(c.tables[0, at // 16]), at % 16][0, 7] = float("inf")
    for max_len in (0, 1):
        out, lse = c.buffers()
        c.operator().run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, lse=lse, max_len=max_len)
        got = oc.wide(out)[0]
        assert np.isposinf(got[:, 7]).all() and np.isfinite(np.delete(got, 7, axis=1)).all()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [4, 64])
@pytest.mark.parametrize("size", ["largest", "smallest"])
def test_means_of_the_types_largest_and_smallest_values(kind, heads, size):
    """Weights that are all alike and some that are not: sums over the tokens that are far beyond what is summed, and
    products with small weights that are normal numbers of 32 bits by a little."""
    lens = [700, 2, 20011, 1]
    c = Case(kind, kind, "flash", lens, heads, 1, 64, 16, seed=36, spread=0.5)
    info = torch.finfo(oc.torch_type(kind))
    most = float(info.max) if size == "largest" else float(info.tiny) * (2.0 ** 17 if kind == "bf16" else 1.0)
    c.q[0] = 0                                               # all weights alike
    v, plain = oc.kv_views("flash", c.cache)[1].view(c.cache_type), c.plain[1]
    for b, n in enumerate(lens):
        t = np.arange(n)
        page = c.tables[b][t // 16].astype(np.int64)
        rows = torch.full((n, 1, 64), most, dtype=c.cache_type, device="cuda")
        rows[:, :, 32:] *= -1
        rows[1::2, :, 16:48] *= 0.5
        v[torch.from_numpy(page).cuda(), torch.from_numpy(t % 16).cuda()] = rows
        plain[page, t % 16] = oc.wide(rows)
    op, exact = c.operator(), c.exact()
    for max_len in (0, 1):
        c.check(op, exact, max_len=max_len)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_every_8_bit_value_is_itself(kind):
    """One token: the output is its row of V, times the scale; NaN included. As keys: scores that are
    the value times a query of one."""
    cache = torch.zeros((1, 1, 2, 1, 256), device="cuda", dtype=torch.uint8)
    cache[0, 0, 1, 0] = torch.arange(256, device="cuda").to(torch.uint8)
    handle = kvt_amd.Cache(0, [[cache]], [512])
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_RAGGED_FLASH, "e4m3", 1, 1, 1, 256)
    op = kvt_amd.DecodeAttention(0, lay, kind, 1, max_seqs=1)
    q, out = (torch.zeros((1, 1, 256), device="cuda", dtype=oc.torch_type(kind)) for _ in range(2))
    table, one = (torch.full(s, v, device="cuda", dtype=torch.int32) for s, v in (((1, 1), 0), ((1,), 1)))
    op.run(handle, 0, q, table, one, out)
    want = oc.wide(cache[0, 0, 1, 0].view(torch.float8_e4m3fn))
    assert np.array_equal(oc.wide(out)[0, 0], want, equal_nan=True)
    op.run(handle, 0, q, table, one, out, v_scale=0.5)
    assert np.array_equal(oc.wide(out)[0, 0], want * 0.5, equal_nan=True)
    # 256 tokens of one dim that counts: lse of each alone is the score
    keys = torch.zeros((256, 1, 2, 1, 16), device="cuda", dtype=torch.uint8)
    keys[:, 0, 0, 0, 3] = torch.arange(256, device="cuda").to(torch.uint8)
    handle = kvt_amd.Cache(0, [[keys]], [keys.numel()])
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_RAGGED_FLASH, "e4m3", 256, 1, 1, 16)
    op = kvt_amd.DecodeAttention(0, lay, kind, 1, max_seqs=256, softmax_scale=1.0)
    q = torch.zeros((256, 1, 16), device="cuda", dtype=oc.torch_type(kind))
    q[:, 0, 3] = 1
    lse = torch.empty((256, 1), device="cuda")
    op.run(handle, 0, q, torch.arange(256, device="cuda", dtype=torch.int32)[:, None],
           torch.ones(256, device="cuda", dtype=torch.int32), torch.empty_like(q), lse=lse)
    got = oc.wide(lse)[:, 0]
    # (log2 e in, ln 2 out: two roundings of 32 bits each)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    held = ~np.isnan(want)
    assert (np.abs(got - want)[held] <= 4 * 2.0 ** -24 * np.abs(want)[held] + 2.0 ** -30).all()


@pytest.mark.parametrize("kind,cache_kind", [("bf16", "bf16"), ("f16", "f16"), ("f16", "e4m3")])
@pytest.mark.parametrize("gap", [4.0, 11.0, 16.0, 20.0, 28.0])
def test_one_token_that_stands_out_of_many(kind, cache_kind, gap):
    """Weights of exp(-gap) against 1, thousands of them: what each is rounded by must not add up."""
    n = 30011
    c = Case(kind, cache_kind, "flash", [n], 4, 1, 64, 16, seed=24)
    where = c.tables[0, np.arange(n) // 16], np.arange(n) % 16
    for view, plain, value in zip(oc.kv_views("flash", c.cache), c.plain, (0.0, 10.0)):
        row = torch.full((64,), value).to(c.cache_type)
        view[torch.from_numpy(where[0]).cuda(), torch.from_numpy(where[1]).cuda()] = row.view(view.dtype).cuda()
        plain[where] = value
    one = int(c.tables[0, 700]), 3
    for view, plain, value in zip(oc.kv_views("flash", c.cache), c.plain, (4.0, 0.0)):
        view[one] = torch.full((1, 64), value).to(c.cache_type).view(view.dtype).cuda()
        plain[one] = value
    c.q.fill_(0)
    c.q[:, :, 5] = gap / 4                                   # (exact in every type)
    exact, op = c.exact(scale=1.0), c.operator(softmax_scale=1.0)
    for max_len in (0, 1):
        c.check(op, exact, max_len=max_len)


def test_long_sequences_split_over_the_device():
    for kind, cache_kind, layout, n, heads, kv, dim, block in (
            ("bf16", "bf16", "flash", 20011, 8, 2, 128, 16), ("f16", "e4m3", "hnd", 33333, 4, 1, 64, 64),
            ("bf16", "bf16", "ragged", 9001, 20, 1, 256, 5)):
        c = Case(kind, cache_kind, layout, [n, 1, 0, n // 2], heads, kv, dim, block, seed=11)
        op, exact = c.operator(), c.exact()
        first = c.check(op, exact)
        for max_len in (n, 1, 4096):
            c.check(op, exact, max_len=max_len)
        for _ in range(5):                                   # whatever order the workgroups end in
            again = c.check(op, exact)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("kind,cache_kind,layout,lens,heads,kv_heads,dim,block", [
    ("bf16", "bf16", "flash", [20011], 64, 1, 128, 16), ("f16", "f16", "hnd", [9001, 0, 7], 33, 1, 256, 16),
    ("bf16", "e4m3", "ragged", [12345, 3000], 128, 2, 64, 5), ("bf16", "bf16", "flash", [33000], 32, 4, 128, 16),
    ("bf16", "bf16", "pages", [1100, 8192], 70, 1, 192, 64)])
def test_many_heads_split_so_far_that_parts_are_joined_in_two_steps(kind, cache_kind, layout, lens, heads, kv_heads, dim,
                                                                    block):
    c = Case(kind, cache_kind, layout, lens, heads, kv_heads, dim, block, seed=25)
    op, exact = c.operator(), c.exact()
    first = c.check(op, exact)
    for max_len in (max(lens), 1, 2000):
        c.check(op, exact, max_len=max_len)
    for _ in range(4):
        again = c.check(op, exact)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def _cut(lens, teams):
    """Of every sequence that is split: (first share, whether that held something before it, number of shares)."""
    units = [-(-n // 128) for n in lens]
    total, before, rows = sum(units), 0, []
    teams = min(teams, total)
    for n in units:
        if n:
            w0, w1 = ((before + 1) * teams - 1) // total, ((before + n) * teams - 1) // total
            if w1 > w0:
                rows.append((w0, w0 * total // teams < before, w1 - w0 + 1))
        before += n
    return rows


@pytest.mark.parametrize("kind,cache_kind,layout,lens,heads,kv_heads,dim,block,shares", [
    ("bf16", "bf16", "flash", [700, 50011, 0, 3000, 41005, 5, 200], 64, 1, 128, 16, 512),
    ("bf16", "e4m3", "hnd", [700, 85027, 33, 9000], 64, 1, 128, 32, 512),
    ("f16", "e4m3", "flash", [700, 155057, 77], 40, 1, 64, 64, 1024),
    ("f16", "f16", "pages", [1300, 150001, 1, 20000], 48, 1, 64, 16, 1024),
    ("bf16", "e4m3", "ragged", [2000, 30007], 64, 2, 256, 16, 128),
    ("f16", "f16", "flash", [1000, 33001, 129, 3000], 33, 1, 256, 48, 256)])
def test_joins_in_two_steps_that_begin_inside_another_sequences_share(kind, cache_kind, layout, lens, heads, kv_heads, dim,
                                                                     block, shares):
    cut = _cut(lens, shares)
    assert any(w0 > 0 and behind and parts > 8 for w0, behind, parts in cut), cut
    c = Case(kind, cache_kind, layout, lens, heads, kv_heads, dim, block, seed=33)
    op, exact = c.operator(), c.exact()
    first = c.check(op, exact)
    c.check(op, exact, max_len=1)                            # (unsplit: the join in one step or none)
    for _ in range(3):
        again = c.check(op, exact)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("kind,cache_kind,heads,kv_heads,dim,shares", [
    ("bf16", "bf16", 64, 4, 128, 256), ("f16", "e4m3", 48, 4, 64, 512), ("bf16", "e4m3", 64, 4, 256, 128),
    ("bf16", "bf16", 96, 6, 128, 170)])
def test_two_heads_side_by_side_joined_in_two_steps(kind, cache_kind, heads, kv_heads, dim, shares):
    """A table with room for far longer sequences makes the launch one for a large batch."""
    lens = [830, 70001, 0, 5000]
    cut = _cut(lens, shares)
    assert any(w0 > 0 and behind and parts > 8 for w0, behind, parts in cut), cut
    c = Case(kind, cache_kind, "flash", lens, heads, kv_heads, dim, 16, seed=34)
    c.tables = np.pad(c.tables, ((0, 0), (0, 20000)), constant_values=-1)
    c.d_tables = torch.from_numpy(c.tables).cuda()
    op, exact = c.operator(), c.exact()
    first = c.check(op, exact)
    c.check(op, exact, max_len=70001)
    for _ in range(3):
        again = c.check(op, exact)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("n", [63, 64, 65, 700])
def test_many_short_sequences(n):
    rng = np.random.default_rng(12)
    c = Case("bf16", "bf16", "flash", rng.integers(0, 70, n), 4, 2, 64, 16, seed=12)
    c.check(c.operator(max_seqs=1000), c.exact(), max_len=70)


def test_uneven_sequences_in_many_shares():
    """More sequences than a wavefront has lanes, one much longer than the rest, empty ones in front,
    between and behind: shares that begin and end anywhere."""
    lens = [0, 0, 5] + [0, 40, 129, 0] * 30 + [9000] + [1, 0, 128] * 25 + [0, 0]
    for kv, heads, dim in ((1, 4, 64), (3, 9, 128)):
        c = Case("bf16", "bf16", "hnd", lens, heads, kv, dim, 16, seed=20)
        op, exact = c.operator(), c.exact()
        first = c.check(op, exact)
        for max_len in (1, 300):
            c.check(op, exact, max_len=max_len)
        again = c.check(op, exact)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("kind,cache_kind,layout,heads,kv_heads,dim,block", [
    ("bf16", "bf16", "flash", 8, 4, 128, 16), ("f16", "f16", "ragged", 20, 4, 80, 5), ("bf16", "e4m3", "pages", 96, 6, 256, 16),
    ("bf16", "bf16", "flash", 4, 4, 64, 16)])
def test_batches_large_enough_to_take_two_heads_side_by_side(kind, cache_kind, layout, heads, kv_heads, dim, block):
    rng = np.random.default_rng(22)
    lens = [int(n) for n in rng.integers(0, 400, 200)] + [0, 1, 2500]
    c = Case(kind, cache_kind, layout, lens, heads, kv_heads, dim, block, seed=22)
    op, exact = c.operator(), c.exact()
    many = c.check(op, exact, max_len=100000)      # as many units as make it worth it, says the caller
    c.check(op, exact, max_len=1)
    again = c.check(op, exact, max_len=100000)
    assert torch.equal(many[0], again[0]) and torch.equal(many[1], again[1])


def test_pages_of_a_cache_beyond_32_bits_that_end_inside_a_tile():
    """Offsets that need 64 bits and block sizes that are no multiple of 16: a cache of 5 GiB."""
    block, kv, dim = 5, 1, 256
    n_blocks = (5 << 30) // (2 * block * kv * dim * 2)
    cache = torch.zeros((n_blocks, 2, block, kv, dim), device="cuda", dtype=torch.bfloat16)
    handle = kvt_amd.Cache(0, [[cache]], [cache.numel() * 2])
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_QWEN3_NEXT_FLASH, "bf16", n_blocks, block, kv, dim)
    g = torch.Generator(device="cuda")
    g.manual_seed(21)
    ids = np.array([n_blocks - 1, 0, n_blocks - 7] + list(range(n_blocks // 2, n_blocks // 2 + 60)), dtype=np.int64)
    n = block * len(ids) - 2
    k, v, q = (torch.randn((m, h, dim), generator=g, device="cuda").to(torch.bfloat16)
               for m, h in ((n, kv), (n, kv), (1, 4)))
    kvt_amd.kv_append(handle, 0, lay, k, v, torch.from_numpy(ids[np.arange(n) // block] * block + np.arange(n) % block).cuda())
    out, lse = torch.empty_like(q), torch.empty((1, 4), device="cuda")
    op = kvt_amd.DecodeAttention(0, lay, "bf16", 4, max_seqs=1)
    op.run(handle, 0, q, torch.from_numpy(ids.astype(np.int32)[None]).cuda(),
           torch.tensor([n], dtype=torch.int32, device="cuda"), out, lse=lse)
    pad = ((0, 2), (0, 0), (0, 0))
    exact = oc.decode_exact(oc.wide(q), *(np.pad(oc.wide(x), pad).reshape(len(ids), block, kv, dim) for x in (k, v)),
                            np.arange(len(ids))[None], [n], block, dim ** -0.5)
    hold(out, lse, exact, "bf16")


@pytest.fixture(scope="module")
def far_bytes():
    """5 GiB in which every element of every type is NaN."""
    return torch.full((5 << 30,), 0xFF, device="cuda", dtype=torch.uint8)


@pytest.mark.parametrize("kind,cache_kind", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("dim,block", [(16, 24), (16, 1), (32, 5), (48, 5), (64, 3), (80, 24), (96, 5), (112, 7), (128, 5),
                                       (144, 24), (192, 5), (240, 3)])
def test_head_sizes_in_a_cache_beyond_32_bits(far_bytes, kind, cache_kind, dim, block):
    """Pages 128 MiB apart that end inside a tile: every row of K and V, of every head size."""
    n_blocks, kv, heads, size = 40, 2, 6, 1 if cache_kind == "e4m3" else 2
    far_bytes.fill_(0xFF)
    handle = kvt_amd.Cache(0, [[far_bytes]], [far_bytes.numel()])
    row = dim * size
    strides = (128 << 20, block * kv * row, kv * row, row)
    lay = kvt_amd.KvLayout(None, cache_kind, n_blocks, block, kv, dim, strides=strides)
    g = torch.Generator(device="cuda")
    g.manual_seed(dim * 100 + block)
    lens = [block * 33 - block // 2, 1, block * 4]
    ids = torch.randperm(n_blocks, generator=g, device="cuda")[:38].split([33, 1, 4])
    tables = np.full((3, 33), -1, dtype=np.int32)
    where = []
    for b, (n, mine) in enumerate(zip(lens, ids)):
        tables[b, :len(mine)] = mine.cpu().numpy()
        t = torch.arange(n, device="cuda")
        where.append(mine[t // block] * block + t % block)
    where = torch.cat(where)
    k, v = (torch.randn((sum(lens), kv, dim), generator=g, device="cuda").to(oc.torch_type(kind)) for _ in range(2))
    q = (2 * torch.randn((3, heads, dim), generator=g, device="cuda")).to(oc.torch_type(kind))
    kvt_amd.kv_append(handle, 0, lay, k, v, where)
    plain, at = [], (where.cpu().numpy() // block, where.cpu().numpy() % block)
    for rows in (k, v):
        pages = np.zeros((n_blocks, block, kv, dim))
        pages[at] = oc.wide(rows.to(oc.torch_type(cache_kind)))
        plain.append(pages)
    out, lse = torch.empty_like(q), torch.empty((3, heads), device="cuda")
    op = kvt_amd.DecodeAttention(0, lay, kind, heads, max_seqs=3)
    exact = oc.decode_exact(oc.wide(q), *plain, tables, lens, block, dim ** -0.5)
    for max_len in (0, 1):
        op.run(handle, 0, q, torch.from_numpy(tables).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), out,
               lse=lse, max_len=max_len)
        hold(out, lse, exact, kind)


def test_offsets_beyond_32_bits():
    """Pages at the far end of a cache of 9 GiB, K and V more than 4 GiB apart."""
    block, kv, dim, n_blocks = 16, 2, 64, 1 << 21
    cache = torch.zeros((2, n_blocks, block, kv, dim), device="cuda", dtype=torch.bfloat16)
    handle = kvt_amd.Cache(0, [[cache]], [cache.numel() * 2])
    lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", n_blocks, block, kv, dim)
    g = torch.Generator(device="cuda")
    g.manual_seed(13)
    ids = np.array([n_blocks - 1, 0, n_blocks - 7, n_blocks // 2 + 1, n_blocks - 3], dtype=np.int64)
    n = 16 * len(ids) - 5
    k, v, q = (torch.randn((m, h, dim), generator=g, device="cuda").to(torch.bfloat16)
               for m, h in ((n, kv), (n, kv), (1, 4)))
    slots = torch.from_numpy(ids[np.arange(n) // block] * block + np.arange(n) % block).cuda()
    kvt_amd.kv_append(handle, 0, lay, k, v, slots)
    at = slots // block, slots % block
    assert torch.equal(cache[0][at], k) and torch.equal(cache[1][at], v)
    out, lse = torch.empty_like(q), torch.empty((1, 4), device="cuda")
    op = kvt_amd.DecodeAttention(0, lay, "bf16", 4, max_seqs=1)
    op.run(handle, 0, q, torch.from_numpy(ids.astype(np.int32)[None]).cuda(),
           torch.tensor([n], dtype=torch.int32, device="cuda"), out, lse=lse)
    pad = ((0, 5), (0, 0), (0, 0))
    exact = oc.decode_exact(oc.wide(q), *(np.pad(oc.wide(x), pad).reshape(len(ids), block, kv, dim) for x in (k, v)),
                            np.arange(len(ids))[None], [n], block, dim ** -0.5)
    hold(out, lse, exact, "bf16")


def test_streams_have_workspaces_of_their_own():
    """One operator, two streams, each held back in turn: split launches that overlap."""
    a = Case("bf16", "bf16", "flash", [3000, 2500], 8, 2, 64, 16, seed=14)
    b = Case("bf16", "bf16", "flash", [2500, 3000], 8, 2, 64, 16, seed=15)
    assert a.n_blocks == b.n_blocks
    op, handles = a.operator(workspaces=2), (a, b)
    exact = [x.exact() for x in handles]
    streams = [checkers.side_stream(), checkers.side_stream()]
    buffers = [[x.buffers() for x in handles] for _ in range(6)]
    torch.cuda.synchronize()
    for turn in range(6):
        with torch.cuda.stream(streams[turn % 2]):
            torch.cuda._sleep(20_000_000)
        for x, st, (out, lse) in zip(handles, streams, buffers[turn]):
            op.run(x.handle, 0, x.q, x.d_tables, x.d_lens, out, lse=lse, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for pair in buffers:
        for (out, lse), e in zip(pair, exact):
            hold(out, lse, e, "bf16")
    # a third stream finds none, until one is given back
    out, lse = a.buffers()
    with pytest.raises(kvt_amd.KvtError) as e:
        op.run(a.handle, 0, a.q, a.d_tables, a.d_lens, out)
    assert e.value.code == ERR_INVALID
    op.release(streams[0].cuda_stream)
    op.run(a.handle, 0, a.q, a.d_tables, a.d_lens, out, lse=lse)
    hold(out, lse, exact[0], "bf16")


def test_one_operator_from_several_threads():
    """Calls of four threads at once, each on a stream of its own, in the order the interpreter gives them."""
    c = Case("bf16", "bf16", "flash", [3000, 20, 700], 8, 2, 64, 16, seed=35)
    op, exact = c.operator(workspaces=4), c.exact()
    streams = [checkers.side_stream() for _ in range(4)]
    buffers = [[c.buffers() for _ in range(25)] for _ in streams]
    torch.cuda.synchronize()

    def work(n):
        for out, lse in buffers[n]:
            op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, lse=lse, stream=streams[n].cuda_stream)

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        list(pool.map(work, range(4)))
    torch.cuda.synchronize()
    one = buffers[0][0]
    hold(*one, exact, "bf16")
    for mine in buffers:
        for out, lse in mine:
            assert torch.equal(out, one[0]) and torch.equal(lse, one[1])


def test_releasing_the_per_thread_stream_gives_back_this_threads_workspace_alone():
    """hipStreamPerThread is one handle for a stream of every thread."""
    per_thread = 2
    c = Case("bf16", "bf16", "flash", [3000, 20], 8, 2, 64, 16, seed=28)
    op, exact = c.operator(workspaces=2), c.exact()
    buffers = [c.buffers() for _ in range(4)]
    torch.cuda.synchronize()

    def launch(n, stream):
        out, lse = buffers[n]
        op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, lse=lse, stream=stream)
        torch.cuda.synchronize()

    def elsewhere(n):
        with concurrent.futures.ThreadPoolExecutor(1) as pool:
            pool.submit(launch, n, per_thread).result()

    elsewhere(0)                                             # another thread's stream takes one workspace
    launch(1, per_thread)                                    # and this thread's the other
    op.release(per_thread)
    launch(2, checkers.side_stream().cuda_stream)            # finds the one that this thread has given back
    with pytest.raises(kvt_amd.KvtError) as e:
        launch(3, checkers.side_stream().cuda_stream)        # and no second one
    assert e.value.code == ERR_INVALID
    for out, lse in buffers[:3]:
        hold(out, lse, exact, "bf16")


def test_graphs_replay_with_new_lengths_and_tables():
    c = Case("bf16", "bf16", "hnd", [2000, 5, 0, 900], 8, 2, 64, 16, seed=16)
    op = c.operator()
    st = checkers.side_stream()
    out, lse = c.buffers()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                       # two graphs of one operator, each with its workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            for _ in range(2):
                op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, lse=lse, max_len=2000,
                       stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    rng = np.random.default_rng(16)
    for turn in range(6):
        lens = [int(x) for x in (rng.integers(0, 2001), rng.integers(0, 6), 0, rng.integers(0, 901))]
        c.lens = lens
        c.d_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        c.q.copy_(torch.randn(c.q.shape, device="cuda"))
        out.fill_(9), lse.fill_(9)
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        hold(out, lse, c.exact(), "bf16")
        eager = c.check(op, c.exact(), max_len=2000)
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])


def test_two_graphs_at_once():
    c = Case("bf16", "bf16", "flash", [6000, 5000], 8, 1, 128, 16, seed=17)
    op, exact = c.operator(), c.exact()
    streams = [checkers.side_stream(), checkers.side_stream()]
    torch.cuda.synchronize()
    made = []
    for st in streams:
        out, lse = c.buffers()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            for _ in range(10):
                op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, lse=lse,
                       stream=torch.cuda.current_stream().cuda_stream)
        made.append((graph, out, lse, st))
    for _ in range(4):
        for graph, out, lse, st in made:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, lse, _ in made:
            hold(out, lse, exact, "bf16")


def test_tables_and_lengths_inside_what_is_written_are_refused():
    c = Case("bf16", "bf16", "flash", [100, 64, 40], 4, 2, 64, 16, seed=30)
    op = c.operator()
    out, lse = c.buffers()
    as_int = out.view(torch.int32).flatten()
    cols = c.tables.shape[1]
    for lens, tables, sums in ((as_int[-3:], c.d_tables, None), (c.d_lens, as_int[5:5 + 3 * cols].view(3, cols), None),
                               (lse.view(torch.int32).flatten()[:3], c.d_tables, lse),
                               (c.d_lens, lse.view(torch.int32).flatten()[-3 * 2:].view(3, 2), lse)):
        with pytest.raises(kvt_amd.KvtError) as e:
            op.run(c.handle, 0, c.q, tables, lens, out, lse=sums)
        assert e.value.code == ERR_INVALID and "shares bytes" in str(e.value)
    c.check(op, c.exact())


def test_scales_of_the_cache_whose_products_leave_32_bits_are_refused():
    c = Case("bf16", "e4m3", "flash", [100, 64], 4, 2, 64, 16, seed=32)
    out, _ = c.buffers()
    for kw, k_scale in ((dict(softmax_scale=1e10), 1e30), (dict(softmax_scale=1.0, logit_cap=1e-20), 1e20)):
        op = c.operator(**kw)
        with pytest.raises(kvt_amd.KvtError) as e:
            op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, k_scale=k_scale)
        assert e.value.code == ERR_INVALID and "32 bits" in str(e.value)
    # large ones that do not
    c.check(c.operator(softmax_scale=1e-20), c.exact(scale=1e-20, k_scale=1e20), k_scale=1e20)
    c.check(c.operator(logit_cap=1e30), c.exact(cap=0.0))
    c.check(c.operator(logit_cap=1e-20, softmax_scale=1e10), c.exact(scale=1e10, cap=1e-20))


def test_refusals():
    c = Case("bf16", "bf16", "flash", [100, 64], 4, 2, 64, 16, seed=18)
    out, lse = c.buffers()

    def refused(code, fn):
        with pytest.raises(kvt_amd.KvtError) as e:
            fn()
        assert e.value.code == code, e.value

    op = c.operator(max_seqs=1)
    refused(ERR_INVALID, lambda: op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, out))
    op = c.operator()
    refused(ERR_OUT_OF_RANGE, lambda: op.run(c.handle, 1, c.q, c.d_tables, c.d_lens, out))
    refused(ERR_INVALID, lambda: op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, k_scale=2.0))
    refused(ERR_INVALID, lambda: op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, c.q))
    refused(ERR_INVALID, lambda: op.run(c.handle, 0, c.q, c.d_tables.cpu(), c.d_lens, out))
    refused(ERR_INVALID, lambda: op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, out[:1].expand(2, 4, 64)))
    small = kvt_amd.Cache(0, [[c.cache]], [c.cache.numel()])
    refused(ERR_OUT_OF_RANGE, lambda: op.run(small, 0, c.q, c.d_tables, c.d_lens, out))
    refused(ERR_INVALID, lambda: op.run(c.handle, 0, c.q, c.d_tables, c.d_lens,
                                        c.cache.view(torch.bfloat16).flatten()[-512:].view(2, 4, 64)))
    for over in (out, c.q, c.cache):
        floats = over.view(torch.float32).flatten()[:8].view(2, 4)
        refused(ERR_INVALID, lambda: op.run(c.handle, 0, c.q, c.d_tables, c.d_lens, out, lse=floats))
    for bad in (dict(q=c.q[:, :3]), dict(q=c.q.half()), dict(block_tables=c.d_tables.long()),
                dict(seq_lens=c.d_lens[:1]), dict(lse=lse.half())):
        args = dict(q=c.q, block_tables=c.d_tables, seq_lens=c.d_lens, out=out)
        args.update(bad)
        with pytest.raises(ValueError):
            op.run(c.handle, 0, **args)
    new = kvt_amd.DecodeAttention
    refused(ERR_UNSUPPORTED, lambda: new(0, c.lay, "f16", 4, 2))
    refused(ERR_UNSUPPORTED, lambda: new(0, c.lay, "f32", 4, 2))
    refused(ERR_INVALID, lambda: new(0, c.lay, "bf16", 3, 2))
    refused(ERR_INVALID, lambda: new(0, c.lay, "bf16", 0, 2))
    refused(ERR_INVALID, lambda: new(0, c.lay, "bf16", 4, 0))
    refused(ERR_INVALID, lambda: new(0, c.lay, "bf16", 4, 65536))
    refused(ERR_INVALID, lambda: new(0, c.lay, "bf16", 4, 2, workspaces=0))
    refused(ERR_INVALID, lambda: new(0, c.lay, "bf16", 4, 2, logit_cap=-1.0))
    refused(ERR_INVALID, lambda: new(0, c.lay, "bf16", 4, 2, softmax_scale=float("nan")))
    refused(ERR_INVALID, lambda: new(99, c.lay, "bf16", 4, 2))
    # no sequences: no launch
    op.run(c.handle, 0, c.q[:0], c.d_tables[:0], c.d_lens[:0], out[:0])
    torch.cuda.synchronize()
    assert (out == 77).all()
