"""The operators on the paged cache as an engine uses them, together with the transfer: prompts
appended to a prefill instance's cache layer by layer, sent by a session, scattered into a decode
instance's cache under other block tables, and tokens decoded there -- each step's query and key
rotated and appended, then attended to. Also from a tensor-parallel bf16 sender to an 8-bit cache.
Held to the formulas in 64 bits on the CPU. Needs a real MI355X."""
import numpy as np
import pytest

import checkers
import kvt_amd
import operator_cases as oc
from kvt_amd import ctypes_defs, pipeline, workloads

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

HEADS, KV, DIM, BLOCK, LAYERS = 8, 2, 128, 16, 3


def _normal(shape, g, kind=torch.bfloat16):
    return torch.randn(shape, generator=g, device="cuda").to(kind)


def _slots(tables, seq, positions):
    t = np.asarray(tables[seq], dtype=np.int64)
    return t[positions // BLOCK] * BLOCK + positions % BLOCK


class Model:
    """What a layer's projections give: rows per (layer, token), kept to compute the answer from."""

    def __init__(self, lens, seed, freq, mag):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)
        self.freq, self.mag = freq, mag
        self.k = [[[] for _ in lens] for _ in range(LAYERS)]     # rotated, in 64 bits and as the cache rounds
        self.v = [[[] for _ in lens] for _ in range(LAYERS)]

    def rows(self, n):
        wide = _normal((n, HEADS + 2 * KV, DIM), self.g)
        return wide[:, :HEADS], wide[:, HEADS:HEADS + KV], wide[:, HEADS + KV:]

    def note(self, layer, seq, cache_rows, v):
        self.k[layer][seq].append(oc.wide(cache_rows))
        self.v[layer][seq].append(oc.wide(v))


def _attention(model, layer, seq, q):
    """(out, lse, measure) of one query [heads, dim] over everything noted."""
    k, v = (np.concatenate(x[layer][seq]) for x in (model.k, model.v))
    pages = k.reshape(1, len(k), KV, DIM), v.reshape(1, len(v), KV, DIM)
    return oc.decode_exact(q[None], *pages, np.zeros((1, 1), dtype=np.int32), [len(k)], len(k), DIM ** -0.5)


@pytest.mark.parametrize("captured", [False, True])
def test_prompts_sent_to_a_decode_instance_and_continued_there(captured):
    lens = [37, 160, 1]
    steps = 20
    freq, mag = kvt_amd.rotary_frequencies(DIM, base=500000.0, scaling="bands", factor=8.0, original_max_position=8192)
    rotary = kvt_amd.Rotary(DIM, frequencies=freq, magnitude=mag)
    model = Model(lens, 1, freq, mag)
    rng = np.random.default_rng(2)
    p_pool, d_pool = 40, 64
    need = [-(-(n + steps) // BLOCK) for n in lens]
    perm = rng.permutation(p_pool)
    p_tables = [perm[i * 12:i * 12 + -(-n // BLOCK)].tolist() for i, n in enumerate(lens)]
    perm, at = rng.permutation(d_pool), 0
    d_tables = []
    for n in need:
        d_tables.append(perm[at:at + n].tolist())
        at += n
    nan = torch.tensor(0x7FC0, dtype=torch.int16, device="cuda")
    p_layers = [[nan.expand(2, p_pool, BLOCK, KV, DIM).contiguous().view(torch.bfloat16)] for _ in range(LAYERS)]
    d_layers = [[nan.expand(2, d_pool, BLOCK, KV, DIM).contiguous().view(torch.bfloat16)] for _ in range(LAYERS)]
    p_bytes, d_bytes = (x[0][0].numel() * 2 for x in (p_layers, d_layers))
    p_cache, d_cache = kvt_amd.Cache(0, p_layers, [p_bytes]), kvt_amd.Cache(0, d_layers, [d_bytes])
    p_lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", p_pool, BLOCK, KV, DIM)
    d_lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", d_pool, BLOCK, KV, DIM)

    # the transfer's plan: the prompts' blocks from the prefill cache to the decode cache
    tok = 2 * KV * DIM * 2
    info = dict(block_sizes=[tok * BLOCK], token_sizes=[tok], num_kv_heads=KV, num_layers=LAYERS)
    src = ctypes_defs.make_worker_info(layer_num_blocks=p_pool, **info)
    dst = ctypes_defs.make_worker_info(layer_num_blocks=d_pool, **info)
    tasks = [ctypes_defs.TaskBuf(0, n, True, [p], [d[:len(p)]]) for n, p, d in zip(lens, p_tables, d_tables)]
    lists, _ = pipeline.parse_batch(ctypes_defs.SHAPE_FLASH, src, dst, tasks)
    plan = kvt_amd.Plan(0, lists, [p_bytes], [d_bytes])
    packed = torch.zeros(LAYERS * plan.layer_bytes, dtype=torch.uint8, device="cuda")
    session = kvt_amd.Session(plan, p_cache, packed, plan.layer_bytes)

    # prefill: all prompts' tokens in one batch, padded; each layer is sent as it is complete
    st = checkers.side_stream()
    total, pad = sum(lens), 7
    slots = np.full(total + pad, -1, dtype=np.int64)
    slots[:total] = np.concatenate([_slots(p_tables, s, np.arange(n)) for s, n in enumerate(lens)])
    pos = np.zeros(total + pad, dtype=np.int64)
    pos[:total] = np.concatenate([np.arange(n) for n in lens])
    d_slots, d_pos = torch.from_numpy(slots).cuda(), torch.from_numpy(pos).cuda()
    inputs = [model.rows(total + pad) for _ in range(LAYERS)]
    torch.cuda.synchronize()
    step = session.begin_step()
    for layer, (q, k, v) in enumerate(inputs):
        kvt_amd.kv_append(p_cache, layer, p_lay, k, v, d_slots, rotary=rotary, positions=d_pos, q=q, q_out=q,
                          stream=st.cuda_stream)
        session.save_layer(layer, st.cuda_stream)
    for layer in range(LAYERS):
        session.wait_layer(layer, step, timeout_us=20_000_000)
    plan.unpack(d_cache, 0, LAYERS, packed, plan.layer_bytes, st.cuda_stream)
    st.synchronize()
    for layer, (_, k, v) in enumerate(inputs):
        exact, scale = oc.rotated(oc.wide(k), pos, freq, mag, DIM, False)
        tol = oc.rotation_tolerance(exact, scale, "bf16")
        first = 0
        for s, n in enumerate(lens):
            where = torch.from_numpy(_slots(d_tables, s, np.arange(n))).cuda()
            got = d_layers[layer][0][0].flatten(0, 1)[where]
            assert (np.abs(oc.wide(got) - exact[first:first + n]) <= tol[first:first + n]).all()
            assert torch.equal(d_layers[layer][0][1].flatten(0, 1)[where], v[first:first + n])
            model.note(layer, s, got, v[first:first + n])
            first += n

    # decode: one batch padded to four sequences, all layers per step
    n_seqs = 4
    attention = kvt_amd.DecodeAttention(0, d_lay, "bf16", HEADS, max_seqs=n_seqs)
    columns = max(need)
    tables = np.full((n_seqs, columns), -1, dtype=np.int32)
    for s, t in enumerate(d_tables):
        tables[s, :len(t)] = t
    d_tab = torch.from_numpy(tables).cuda()
    seq_lens = torch.zeros(n_seqs, dtype=torch.int32, device="cuda")
    slots_in, pos_in = (torch.zeros(n_seqs, dtype=torch.int64, device="cuda") for _ in range(2))
    qkv = [torch.zeros((n_seqs, HEADS + 2 * KV, DIM), dtype=torch.bfloat16, device="cuda") for _ in range(LAYERS)]
    q_rot = [torch.zeros((n_seqs, HEADS, DIM), dtype=torch.bfloat16, device="cuda") for _ in range(LAYERS)]
    outs = [torch.zeros_like(q_rot[0]) for _ in range(LAYERS)]
    lses = [torch.zeros((n_seqs, HEADS), device="cuda") for _ in range(LAYERS)]

    def forward(stream):
        for layer in range(LAYERS):
            x = qkv[layer]
            kvt_amd.kv_append(d_cache, layer, d_lay, x[:, HEADS:HEADS + KV], x[:, HEADS + KV:], slots_in, rotary=rotary,
                              positions=pos_in, q=x[:, :HEADS], q_out=q_rot[layer], stream=stream)
            attention.run(d_cache, layer, q_rot[layer], d_tab, seq_lens, outs[layer], lse=lses[layer],
                          max_len=columns * BLOCK, stream=stream)

    graph = None
    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            forward(torch.cuda.current_stream().cuda_stream)
    now = np.array(lens + [0])
    for turn in range(steps):
        live = now > 0
        slots_h = np.array([_slots(d_tables, s, np.array([now[s]]))[0] if live[s] else -1 for s in range(n_seqs)])
        slots_in.copy_(torch.from_numpy(slots_h))
        pos_in.copy_(torch.from_numpy(now))
        seq_lens.copy_(torch.from_numpy(np.where(live, now + 1, 0).astype(np.int32)))
        for x in qkv:
            x.copy_(_normal(x.shape, model.g))
        torch.cuda.synchronize()
        if captured:
            with torch.cuda.stream(st):
                graph.replay()
        else:
            forward(st.cuda_stream)
        st.synchronize()
        for layer in range(LAYERS):
            x = qkv[layer]
            for s in range(3):
                where = int(slots_h[s])
                got_k = d_layers[layer][0][0].flatten(0, 1)[where:where + 1]
                exact, scale = oc.rotated(oc.wide(x[s:s + 1, HEADS:HEADS + KV]), now[s:s + 1], freq, mag, DIM, False)
                assert (np.abs(oc.wide(got_k) - exact) <= oc.rotation_tolerance(exact, scale, "bf16")).all()
                model.note(layer, s, got_k, x[s:s + 1, HEADS + KV:])
                eo, el, measure = _attention(model, layer, s, oc.wide(q_rot[layer])[s])
                to, tl = oc.decode_tolerance(eo, el, measure, "bf16")
                assert (np.abs(oc.wide(outs[layer])[s] - eo[0]) <= to[0]).all(), (turn, layer, s)
                assert (np.abs(oc.wide(lses[layer])[s] - el[0]) <= tl[0]).all(), (turn, layer, s)
            assert not outs[layer][3].any() and torch.isneginf(lses[layer][3]).all()
        now = np.where(live, now + 1, 0)


def test_bf16_ranks_sent_to_an_8_bit_cache_and_attended_to_there():
    """Two tensor-parallel senders with half the KV heads each; the converting plan's bytes are those
    that an append to the 8-bit cache with scales of 1 would have written for V."""
    kv, dim, heads = 4, 64, 16
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    make = lambda r: workloads.tp_split("flash", 2, 1, r, n_layers=1, src_pool=64, dst_pool=64, n_req=3, min_tok=20,  # noqa: E731
                                        max_tok=200, total_heads=kv, head_dim=dim, fp8_dst=True)
    w = make(0)
    lens = [t[1] for t in w.tasks]
    dst = torch.full((2, 64, 16, kv, dim), 0x7F, dtype=torch.uint8, device="cuda")
    direct = dst.clone()
    d_cache = kvt_amd.Cache(0, [[dst]], [dst.numel()])
    direct_cache = kvt_amd.Cache(0, [[direct]], [direct.numel()])
    rotary = kvt_amd.Rotary(dim)
    freq, mag = kvt_amd.rotary_frequencies(dim)
    n = sum(lens)
    k, v = (_normal((n, kv, dim), g) for _ in range(2))
    pos = np.concatenate([np.arange(m) for m in lens])
    d_pos = torch.from_numpy(pos).cuda()
    tables = {side: [t[3 if side == "src" else 4][0] for t in w.tasks] for side in ("src", "dst")}
    slots = {side: torch.from_numpy(np.concatenate([_slots(t, s, np.arange(m)) for s, m in enumerate(lens)])).cuda()
             for side, t in tables.items()}
    for rank in (0, 1):
        w = make(rank)
        src = torch.zeros((2, 64, 16, kv // 2, dim), dtype=torch.bfloat16, device="cuda")
        s_cache = kvt_amd.Cache(0, [[src]], [src.numel() * 2])
        lay = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "bf16", 64, 16, kv // 2, dim)
        mine = slice(rank * kv // 2, (rank + 1) * kv // 2)
        kvt_amd.kv_append(s_cache, 0, lay, k[:, mine], v[:, mine], slots["src"], rotary=rotary, positions=d_pos)
        plan, _ = pipeline.build_plan_runs(w, 0)
        packed = torch.zeros(plan.layer_bytes, dtype=torch.uint8, device="cuda")
        plan.pack(s_cache, 0, 1, packed, plan.layer_bytes)
        plan.unpack(d_cache, 0, 1, packed, plan.layer_bytes)
    lay8 = kvt_amd.KvLayout(kvt_amd.SHAPE_FLASH, "e4m3", 64, 16, kv, dim)
    kvt_amd.kv_append(direct_cache, 0, lay8, k, v, slots["dst"], rotary=rotary, positions=d_pos)
    torch.cuda.synchronize()
    rows = [x.flatten(1, 2)[:, slots["dst"]] for x in (dst, direct)]
    assert torch.equal(rows[0][1], rows[1][1])
    # K went through bf16 on the way: within that rounding and one to e4m3 of the formula
    exact, scale = oc.rotated(oc.wide(k), pos, freq, mag, dim, False)
    sent = oc.wide(rows[0][0].view(torch.float8_e4m3fn))
    via = oc.rotation_tolerance(exact, scale, "bf16")
    assert (np.abs(sent - exact) <= via + oc.HALF_STEP["e4m3"][0] * (np.abs(exact) + via) + oc.HALF_STEP["e4m3"][1]).all()
    tab = np.full((3, max(len(t) for t in tables["dst"])), -1, dtype=np.int32)
    for s, t in enumerate(tables["dst"]):
        tab[s, :len(t)] = t
    q = (2 * torch.randn((3, heads, dim), generator=g, device="cuda")).to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty((3, heads), device="cuda")
    attention = kvt_amd.DecodeAttention(0, lay8, "bf16", heads, max_seqs=3)
    attention.run(d_cache, 0, q, torch.from_numpy(tab).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), out,
                  lse=lse)
    pages = [np.nan_to_num(oc.wide(x.view(torch.float8_e4m3fn))) for x in (dst[0], dst[1])]
    eo, el, measure = oc.decode_exact(oc.wide(q), *pages, tab, lens, 16, dim ** -0.5)
    to, tl = oc.decode_tolerance(eo, el, measure, "bf16")
    assert (np.abs(oc.wide(out) - eo) <= to).all() and (np.abs(oc.wide(lse) - el) <= tl).all()
