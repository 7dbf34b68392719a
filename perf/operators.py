"""What is measured of the operators on the paged cache, next to the transfer of its pages: rotary
positions, appending a step's keys and values to the cache (rotated on the way), and the attention
of one new token over it.

`run` computes them in plain torch operations in 32 bits (angles in 64), or, where `own` is set,
by the calls that an engine makes of kvt_amd. A case is a dict of plain values:

  op        "rotary" | "append" | "decode"
  dtype     of queries, keys and values: "bf16" | "f16" | "f32" (f32: rotary alone)
  cache     element type of the cache: "bf16" | "f16" | "e4m3"
  layout    "flash" [2, nblk, bs, h, d] | "ragged" [nblk, bs, 2, h, d] | "hnd" [nblk, 2, h, bs, d]
            | "pages" [nblk, 2, bs, h, d]
  heads, kv_heads, dim, block (tokens per cache block)
  tokens    of a rotary or append call; seqs, min_len, max_len of a decode call
"""
import math
import random
import sys

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}


# ------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decode step of 64 requests: the query and key heads of a fused projection
        dict(name="rotary step 64", op="rotary", dtype="bf16", tokens=64, heads=40, kv_heads=8, dim=128,
             rotary_dim=128, interleaved=False, base=500000.0, scaling="bands", factor=8.0, original=8192,
             max_pos=131072),
        # a long prompt of a wide model, interleaved pairs
        dict(name="rotary prompt interleaved", op="rotary", dtype="f16", tokens=16384, heads=64, kv_heads=8,
             dim=128, rotary_dim=128, interleaved=True, base=10000.0, scaling="none", factor=1.0, original=0,
             max_pos=16384),
        # far positions, a quarter of a wide head, in 32 bits
        dict(name="rotary far f32 partial", op="rotary", dtype="f32", tokens=4099, heads=18, kv_heads=2, dim=256,
             rotary_dim=64, interleaved=False, base=1000000.0, scaling="ramp", factor=32.0, original=32768,
             max_pos=1048576),
        # one request's decode step: what counts is the call itself
        dict(name="append one token", op="append", dtype="bf16", cache="bf16", layout="flash", tokens=1, padded=0,
             heads=32, kv_heads=8, dim=128, block=16, rotary_dim=128, interleaved=False, base=500000.0,
             scaling="bands", factor=8.0, original=8192, max_pos=131072, blocks=1024),
        # a decode step of a full batch padded to a captured size, HND pages
        dict(name="append step hnd", op="append", dtype="f16", cache="f16", layout="hnd", tokens=256, padded=19,
             heads=64, kv_heads=8, dim=128, block=16, rotary_dim=128, interleaved=False, base=500000.0,
             scaling="none", factor=1.0, original=0, max_pos=8192, blocks=1024),
        # a prefill step: two prompts of 8192 tokens
        dict(name="append prompt", op="append", dtype="bf16", cache="bf16", layout="flash", tokens=16384, padded=0,
             heads=32, kv_heads=8, dim=128, block=16, rotary_dim=128, interleaved=False, base=500000.0,
             scaling="bands", factor=8.0, original=8192, max_pos=16384, blocks=1280),
        # a prefill step of a hybrid model into an 8-bit cache, an odd number of tokens, a part of the head rotated
        dict(name="append prompt e4m3 partial", op="append", dtype="bf16", cache="e4m3", layout="ragged",
             tokens=10007, padded=7, heads=16, kv_heads=2, dim=256, block=64, rotary_dim=64, interleaved=False,
             base=10000000.0, scaling="linear", factor=4.0, original=0, max_pos=262144, blocks=192),
        # one short request: latency
        dict(name="decode one short", op="decode", dtype="bf16", cache="bf16", layout="flash", seqs=1, min_len=512,
             max_len=512, edge=False, lens=1, heads=32, kv_heads=8, dim=128, block=16, window=0, cap=0.0),
        # one very long request, HND pages: the work of few heads split over the device
        dict(name="decode one long hnd", op="decode", dtype="bf16", cache="bf16", layout="hnd", seqs=1,
             min_len=131071, max_len=131071, edge=False, lens=2, heads=64, kv_heads=8, dim=128, block=16, window=0,
             cap=0.0),
        # 64 requests of 1k to 8k tokens
        dict(name="decode batch ragged", op="decode", dtype="bf16", cache="bf16", layout="flash", seqs=64,
             min_len=1024, max_len=8192, edge=False, lens=20252, heads=32, kv_heads=8, dim=128, block=16, window=0,
             cap=0.0),
        # 128 requests of 4096 tokens, 2 key-value heads of 256
        dict(name="decode pages 256 f16", op="decode", dtype="f16", cache="f16", layout="pages", seqs=128,
             min_len=4096, max_len=4096, edge=False, lens=4, heads=16, kv_heads=2, dim=256, block=16, window=0,
             cap=0.0),
        # an 8-bit cache on one rank of a tensor-parallel instance, empty and one-token rows among long ones
        dict(name="decode e4m3 uneven", op="decode", dtype="bf16", cache="e4m3", layout="ragged", seqs=96,
             min_len=1, max_len=16384, edge=True, lens=5, heads=16, kv_heads=2, dim=128, block=64, window=0,
             cap=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "decode", "decode"])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 160, 192, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16] if op != "decode" else [1, 2, 4, 5, 7, 8, 12, 16, 24, 32])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16"]), heads=kv_heads * group, kv_heads=kv_heads, dim=dim)
    if op != "decode":
        half = rng.choice([dim // 2, dim // 2, dim // 4, dim // 8 + 3])
        c.update(rotary_dim=2 * half, interleaved=rng.random() < 0.4,
                 base=rng.choice([10000.0, 500000.0, 1000000.0]),
                 scaling=rng.choice(["none", "linear", "bands", "ramp"]), factor=rng.choice([2.0, 8.0, 40.0]),
                 original=rng.choice([4096, 8192, 32768]), max_pos=_log(rng, 1000, 1000000))
        row = c["heads"] + 2 * kv_heads
        most = 16384 * 48 * 128 // (row * dim)
        c["tokens"] = _log(rng, 1, most)
    if op == "rotary":
        c["dtype"] = rng.choice(["bf16", "f16", "f32"])
        c["tokens"] = max(1, c["tokens"] // (2 if c["dtype"] == "f32" else 1))
        return c
    c["cache"] = rng.choice([c["dtype"], c["dtype"], "e4m3"])
    c["layout"] = rng.choice(["flash", "ragged", "hnd", "pages"])
    c["block"] = rng.choice([1, 5, 8, 16, 16, 16, 24, 32, 64, 128, 544])
    if op == "append":
        c["padded"] = rng.choice([0, 0, c["tokens"] // 3])
        c["blocks"] = c["tokens"] // c["block"] + rng.randrange(2, 40)
        return c
    c["seqs"] = _log(rng, 1, 192)
    row = 2 * kv_heads * dim * _BYTES[c["cache"]]
    c["max_len"] = min(131071, _log(rng, 1, max(2, (700 << 20) // (row * c["seqs"]))))
    c["min_len"] = rng.choice([1, c["max_len"] // 3 + 1, c["max_len"]])
    c["edge"] = c["seqs"] >= 3 and rng.random() < 0.3
    c["lens"] = rng.randrange(1 << 30)
    c["window"] = rng.choice([0, 0, 0, c["max_len"] // 2 + 1])
    c["cap"] = rng.choice([0.0, 0.0, 0.0, 30.0])
    return c


def _lens(c):
    """The requests' lengths: of the case, so that work() knows them."""
    r = random.Random(c["lens"])
    lens = [r.randint(c["min_len"], c["max_len"]) for _ in range(c["seqs"])]
    if c["edge"]:
        lens[:3] = [0, 1, c["max_len"]]
    return lens


def work(case):
    c = case
    if c["op"] == "rotary":
        x = c["tokens"] * c["heads"] * c["dim"] * _BYTES[c["dtype"]]
        return {"bytes": 2 * x + 8 * c["tokens"], "flops": 3 * c["tokens"] * c["heads"] * c["rotary_dim"]}
    if c["op"] == "append":
        t, live = c["tokens"], c["tokens"] - c["padded"]
        q, kv = t * c["heads"] * c["dim"], 2 * live * c["kv_heads"] * c["dim"]
        return {"bytes": (2 * q + kv) * _BYTES[c["dtype"]] + kv * _BYTES[c["cache"]] + 16 * t,
                "flops": 3 * c["rotary_dim"] * (t * c["heads"] + live * c["kv_heads"])}
    seen = sum(min(n, c["window"]) if c["window"] else n for n in _lens(c))
    q = c["seqs"] * c["heads"] * c["dim"] * _BYTES[c["dtype"]]
    table = sum(-(-n // c["block"]) for n in _lens(c)) * 4
    return {"bytes": 2 * seen * c["kv_heads"] * c["dim"] * _BYTES[c["cache"]] + 2 * q + 4 * c["seqs"] * c["heads"] + table,
            "flops": 4 * seen * c["heads"] * c["dim"]}


# -------------------------------------------------------------------------------- the inputs

_SHAPES = {"flash": lambda n, b, h, d: (2, n, b, h, d), "ragged": lambda n, b, h, d: (n, b, 2, h, d),
           "hnd": lambda n, b, h, d: (n, 2, h, b, d), "pages": lambda n, b, h, d: (n, 2, b, h, d)}


def _new_cache(c, n_blocks, gen):
    """One layer's cache with a history in it."""
    shape = _SHAPES[c["layout"]](n_blocks, c["block"], c["kv_heads"], c["dim"])
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
    return x.to(_TYPES[c["cache"]])


def _kv_views(c, cache):
    """(keys, values) of the cache as [n_blocks, block, h, d] views."""
    if c["layout"] == "flash":
        return cache[0], cache[1]
    if c["layout"] == "ragged":
        return cache[:, :, 0], cache[:, :, 1]
    if c["layout"] == "hnd":
        return cache[:, 0].permute(0, 2, 1, 3), cache[:, 1].permute(0, 2, 1, 3)
    return cache[:, 0], cache[:, 1]


def _frequencies(c):
    """Radians per position of every pair, and what the rotated values are multiplied with."""
    d, f = c["rotary_dim"], c["factor"]
    i = np.arange(d // 2, dtype=np.float64)
    w = c["base"] ** (-2.0 * i / d)
    if c["scaling"] == "linear":
        return w / f, 1.0
    if c["scaling"] == "bands":      # wavelengths up to original / 4 stay, from original / 1 on they grow by f
        turns = c["original"] * w / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return w * keep + w / f * (1 - keep), 1.0
    if c["scaling"] == "ramp":       # a ramp over the pair's number, between 32 turns and one
        at = lambda turns: d * math.log(c["original"] / (turns * 2 * math.pi)) / (2 * math.log(c["base"]))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
        keep = 1 - np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        return w * keep + w / f * (1 - keep), 0.1 * math.log(f) + 1.0
    return w, 1.0


def _positions(c, gen):
    return torch.randint(0, c["max_pos"], (c["tokens"],), generator=gen, device="cuda")


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case=c)
    dt = _TYPES[c["dtype"]]
    if c["op"] in ("rotary", "append"):
        freq, s["magnitude"] = _frequencies(c)
        s["freq"] = torch.from_numpy(freq).cuda()
        s["positions"] = _positions(c, gen)
    if c["op"] == "rotary":
        # the rotated heads are the front part of a fused projection's output
        wide = torch.randn((c["tokens"], c["heads"] + c["kv_heads"], c["dim"]), generator=gen, device="cuda", dtype=dt)
        s["x"] = wide[:, :c["heads"]]
        s["out"] = torch.empty((c["tokens"], c["heads"], c["dim"]), device="cuda", dtype=dt)
    elif c["op"] == "append":
        h, k = c["heads"], c["kv_heads"]
        wide = torch.randn((c["tokens"], h + 2 * k, c["dim"]), generator=gen, device="cuda", dtype=dt)
        s["q"], s["k"], s["v"] = wide[:, :h], wide[:, h:h + k], wide[:, h + k:]
        s["q_out"] = torch.empty((c["tokens"], h, c["dim"]), device="cuda", dtype=dt)
        s["cache"] = _new_cache(c, c["blocks"], gen)
        # whole blocks in the order a paged allocator hands them out, the last rows of the batch padding
        blocks = torch.randperm(c["blocks"], generator=gen, device="cuda")
        t = torch.arange(c["tokens"], device="cuda")
        slots = blocks[t // c["block"]] * c["block"] + t % c["block"]
        slots[c["tokens"] - c["padded"]:] = -1
        s["slots"] = slots
    else:
        lens = _lens(c)
        pages = [-(-n // c["block"]) for n in lens]
        n_blocks = sum(pages) + 3
        s["cache"] = _new_cache(c, n_blocks, gen)
        # queries two and a half times as wide as the keys: some positions stand out, most do not
        s["q"] = (2.5 * torch.randn((c["seqs"], c["heads"], c["dim"]), generator=gen, device="cuda")).to(dt)
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        starts = torch.from_numpy(np.cumsum([0] + pages)[:-1]).cuda()
        p = torch.arange(max(max(pages), 1), device="cuda")
        blocks = torch.randperm(n_blocks, generator=gen, device="cuda")
        held = p < torch.tensor(pages, device="cuda")[:, None]
        s["tables"] = torch.where(held, blocks[torch.where(held, starts[:, None] + p, 0)], 0).to(torch.int32)
        s["out"] = torch.empty((c["seqs"], c["heads"], c["dim"]), device="cuda", dtype=dt)
        s["lse"] = torch.empty((c["seqs"], c["heads"]), device="cuda", dtype=torch.float32)
        s["scale"] = c["dim"] ** -0.5
    if own:
        _handles(c, s)
    return s


def _handles(c, s):
    """What an engine keeps for as long as it runs."""
    if "llumnix-kv_amd" not in sys.path:
        sys.path.insert(0, "llumnix-kv_amd")
    import kvt_amd

    if c["op"] != "decode":
        s["rotary"] = kvt_amd.Rotary(c["rotary_dim"], interleaved=c["interleaved"], frequencies=_frequencies(c)[0],
                                     magnitude=s["magnitude"])
    if c["op"] == "rotary":
        return
    shape = {"flash": kvt_amd.SHAPE_FLASH, "ragged": kvt_amd.SHAPE_RAGGED_FLASH, "hnd": kvt_amd.SHAPE_FLASHINFER,
             "pages": kvt_amd.SHAPE_QWEN3_NEXT_FLASH}[c["layout"]]
    n_blocks = s["cache"].shape[1 if c["layout"] == "flash" else 0]
    s["layout"] = kvt_amd.KvLayout(shape, c["cache"], n_blocks, c["block"], c["kv_heads"], c["dim"])
    s["handle"] = kvt_amd.Cache(0, [[s["cache"]]], [s["cache"].numel() * s["cache"].element_size()])
    if c["op"] == "append":
        s["append"] = kvt_amd.kv_append
    else:
        s["attention"] = kvt_amd.DecodeAttention(0, s["layout"], c["dtype"], c["heads"], max_seqs=c["seqs"],
                                                 softmax_scale=s["scale"], logit_cap=c["cap"], window=c["window"])


# ------------------------------------------------------------------------------- one pass

def run(state):
    return {"rotary": _run_rotary, "append": _run_append, "decode": _run_decode}[state["case"]["op"]](state)


def _cos_sin(s):
    """[tokens, 1, pairs] in 32 bits, from angles in 64."""
    angle = s["positions"].double()[:, None] * s["freq"]
    return tuple((f(angle) * s["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))


def _rotated(c, x, cos, sin):
    """x [tokens, heads, dim] in 32 bits with its first rotary_dim values rotated."""
    x = x.float()
    d = c["rotary_dim"]
    a, b = (x[..., 0:d:2], x[..., 1:d:2]) if c["interleaved"] else (x[..., :d // 2], x[..., d // 2:d])
    p, q = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((p, q), -1).flatten(-2) if c["interleaved"] else torch.cat((p, q), -1)
    return torch.cat((y, x[..., d:]), -1)


def _run_rotary(s):
    c = s["case"]
    if own:
        s["rotary"].apply(s["x"], s["positions"], s["out"])
    else:
        s["out"].copy_(_rotated(c, s["x"], *_cos_sin(s)))
    return s["out"]


def _rounded(c, x):
    """x as the cache holds it, as whole numbers of the cache's width."""
    if c["cache"] == "e4m3":
        return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return x.to(_TYPES[c["cache"]]).view(torch.int16)


def _run_append(s):
    c = s["case"]
    if own:
        s["append"](s["handle"], 0, s["layout"], s["k"], s["v"], s["slots"], rotary=s["rotary"],
                    positions=s["positions"], q=s["q"], q_out=s["q_out"])
    else:
        cos, sin = _cos_sin(s)
        s["q_out"].copy_(_rotated(c, s["q"], cos, sin))
        keep = s["slots"] >= 0
        slots = s["slots"][keep]
        at = (slots // c["block"], slots % c["block"])
        bits = s["cache"].view(torch.uint8 if c["cache"] == "e4m3" else torch.int16)
        keys, values = _kv_views(c, bits)
        keys[at] = _rounded(c, _rotated(c, s["k"], cos, sin)[keep])
        values[at] = _rounded(c, s["v"].float()[keep])
    return {"cache": s["cache"], "q": s["q_out"]}


def _gathered(c, view, tables):
    """[seqs, kv_heads, positions, dim] in 32 bits of a [n_blocks, block, h, d] view."""
    bits = view.view(torch.uint8 if c["cache"] == "e4m3" else torch.int16)
    pages = bits[tables.long()].flatten(1, 2).view(_TYPES[c["cache"]])
    return pages.float().permute(0, 2, 1, 3).contiguous()


def _run_decode(s):
    c = s["case"]
    if own:
        s["attention"].run(s["handle"], 0, s["q"], s["tables"], s["seq_lens"], s["out"], lse=s["lse"],
                           max_len=c["max_len"])
        return {"out": s["out"], "lse": s["lse"]}
    keys, values = (_gathered(c, v, s["tables"]) for v in _kv_views(c, s["cache"]))
    q = s["q"].float().view(c["seqs"], c["kv_heads"], -1, c["dim"])
    score = (q @ keys.transpose(-1, -2).contiguous()) * s["scale"]
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    t = torch.arange(score.shape[-1], device="cuda")
    n = s["seq_lens"][:, None]
    seen = (t < n) & (t >= n - c["window"]) if c["window"] else t < n
    seen = seen[:, None, None]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.where(seen, torch.exp(score - top), 0.0)
    total = weight.sum(-1, keepdim=True)
    out = torch.where(total > 0, (weight / total) @ values, 0.0)
    s["out"].copy_(out.view(s["out"].shape))
    s["lse"].copy_((top + torch.log(total)).view(s["lse"].shape))
    return {"out": s["out"], "lse": s["lse"]}


# ------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    c, s = case, prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "decode": _exact_decode}[c["op"]](c, s)


def _turned(c, s, x):
    """Each pair as a complex number, turned by its angle."""
    y = x.double().clone()
    d = c["rotary_dim"]
    turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["freq"]))[:, None]
    first, second = (slice(0, d, 2), slice(1, d, 2)) if c["interleaved"] else (slice(0, d // 2), slice(d // 2, d))
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rotary(c, s):
    return _turned(c, s, s["x"])


def _exact_append(c, s):
    cache = s["cache"].to(torch.float32).double()
    live = s["slots"] >= 0
    slots = s["slots"][live]
    for view, rows in zip(_kv_views(c, cache), (_turned(c, s, s["k"]), s["v"].double())):
        view[slots // c["block"], slots % c["block"]] = rows[live]
    return {"cache": cache, "q": _turned(c, s, s["q"])}


def _exact_decode(c, s):
    keys, values = _kv_views(c, s["cache"])
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    group = c["heads"] // c["kv_heads"]
    for b, n in enumerate(_lens(c)):
        if n == 0:
            continue
        t = torch.arange(max(0, n - c["window"]) if c["window"] else 0, n, device="cuda")
        at = (s["tables"][b].long()[t // c["block"]], t % c["block"])
        for h in range(c["kv_heads"]):
            mine = slice(h * group, (h + 1) * group)
            k, v = (x[:, :, h][at].to(torch.float32).double() for x in (keys, values))
            z = (s["q"][b, mine].double() @ k.T) * s["scale"]
            if c["cap"]:
                z = c["cap"] * torch.tanh(z / c["cap"])
            lse[b, mine] = torch.logsumexp(z, -1)
            out[b, mine] = torch.softmax(z, -1) @ v
    return {"out": out, "lse": lse}
