"""Rotary positions, an 8-bit key/value cache and attention over it, as measurable cases.

Each case can be run in two forms on the same inputs: with ``own`` false the
operator written out in elementary torch operations, with ``own`` true the
framework's calls (`needle_hip.Rope`, `needle_hip.KvCache8`).

Rotation: pair i of a head's first 2 n dims, (i, i + n) or (2 i, 2 i + 1), turns by
position * frequency_i; cosine and sine, times the plan's amplitude, are rounded
to f32, the products and their sum too.

The cache holds keys and values as whole numbers -127 .. 127 times a step for
each block of 16 positions and head, all in f32: step = max|x| / 127 of the
block's first rows; rows that join a block double its step until it is their
own max|x| / 127 at least, and the numbers that were there are divided by as
much (ties to even).

Kinds:
  rope    rows of queries and keys turned to their positions, or gradients turned back
  store   new rows of every sequence into the cache, keys and queries turned first, and
          the blocks that the rows are in read back
  attend  attention of each sequence's last rows over its 8-bit cache, with first positions
          that stay visible (sink) and a window of last ones (ring; 0: all)
  cross   attention of a decoder's rows to all positions that a sequence's encoder left
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 16


def listed():
    agent = {"kv": 2, "qk": 48, "v": 64, "page": 64, "type": "f32"}
    wide = {"kv": 8, "qk": 128, "v": 128, "page": 64}
    return [
        # One decoding step of eight conversations at the published model's head
        # shapes: launches and host time count.
        {"name": "rope_step", "kind": "rope", "rows": 8, "heads": 12, "kv": 2, "dim": 48, "turned": 48, "layout": "half",
         "theta": 10000.0, "scaling": "none", "first": 300, "back": False, "type": "f32"},
        # A batch of prompts of a wider model whose context was stretched eight times.
        {"name": "rope_prompts", "kind": "rope", "rows": 6001, "heads": 32, "kv": 8, "dim": 128, "turned": 128,
         "layout": "half", "theta": 500000.0, "scaling": "bands", "first": 0, "back": False, "type": "bf16"},
        # The gradients of a training step on a very long text, neighbours paired,
        # a third of each head turned.
        {"name": "rope_back", "kind": "rope", "rows": 4096, "heads": 24, "kv": 24, "dim": 96, "turned": 32,
         "layout": "interleaved", "theta": 10000.0, "scaling": "parts", "first": 990000, "back": True, "type": "f16"},
        # One decoding step of eight conversations: a layer's new rows.
        {"name": "store_step", "kind": "store", "seqs": 8, "rows": 1, "len": 300, "heads": 12, "turned": 48, **agent},
        # Prompts of several requests into one layer of a wider model.
        {"name": "store_prompts", "kind": "store", "seqs": 3, "rows": 2500, "len": 77, "heads": 32, "turned": 128, **wide,
         "type": "bf16"},
        # A decoding step of one agent turn under its span of 118 + 256 positions.
        {"name": "step_agent", "kind": "attend", "seqs": 1, "rows": 1, "len": 700, "heads": 12, "sink": 118, "ring": 256,
         **agent},
        # A server's decoding step: 64 conversations of up to 8192 positions.
        {"name": "step_batch", "kind": "attend", "seqs": 64, "rows": 1, "len": 8192, "heads": 32, "sink": 0, "ring": 0,
         **wide, "type": "bf16"},
        # One conversation over a very long document.
        {"name": "step_document", "kind": "attend", "seqs": 1, "rows": 1, "len": 131072, "heads": 32, "sink": 0,
         "ring": 0, **wide, "type": "f16"},
        # The check of four drafted tokens in 16 conversations, windowed layers.
        {"name": "drafts_window", "kind": "attend", "seqs": 16, "rows": 5, "len": 5000, "heads": 32, "sink": 4,
         "ring": 1024, **wide, "type": "bf16"},
        # A chunk of two long prompts: the queries of 2000 positions after 6000.
        {"name": "prompt_chunk", "kind": "attend", "seqs": 2, "rows": 2000, "len": 8000, "heads": 32, "sink": 0,
         "ring": 0, **wide, "type": "bf16"},
        # A decoding step of four hypotheses each for 16 inputs, one of them without a state.
        {"name": "cross_step", "kind": "cross", "seqs": 16, "rows": 4, "len": 1500, "heads": 16, "empty": True, "kv": 16,
         "qk": 64, "v": 64, "page": 128, "type": "f16"},
        # The decoder's own prompts against its encoder's states.
        {"name": "cross_prompts", "kind": "cross", "seqs": 4, "rows": 448, "len": 1500, "heads": 16, "empty": False,
         "kv": 16, "qk": 64, "v": 64, "page": 128, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _shape(rng):
    """Heads, head widths, page and type of a drawn case."""
    qk, v = rng.choice(((48, 64), (64, 64), (80, 80), (96, 96), (128, 128), (128, 128), (192, 128), (256, 256), (45, 51)))
    return {"kv": rng.choice((1, 2, 3, 4, 8)), "qk": qk, "v": v, "page": rng.choice((64, 128, 256)),
            "type": rng.choice(("f32", "bf16", "bf16", "f16"))}


def draw(rng):
    """One more case of the listed ones' ranges."""
    kind = rng.choice(("rope", "rope", "store", "store", "attend", "attend", "attend", "attend", "cross", "cross"))
    s = _shape(rng)
    if kind == "rope":
        kv, dim = rng.choice((1, 2, 3, 8, 24)), s["qk"]
        heads = kv * rng.choice((1, 2, 4))
        return {"kind": kind, "rows": _log(rng, 1, 6000 * 40 * 128 // ((heads + kv) * dim)), "heads": heads, "kv": kv,
                "dim": dim, "turned": 2 * rng.randrange(1, dim // 2 + 1) if rng.random() < 0.5 else dim // 2 * 2,
                "layout": rng.choice(("half", "interleaved")), "theta": rng.choice((10000.0, 500000.0, 1000000.0)),
                "scaling": rng.choice(("none", "linear", "base", "parts", "bands")),
                "first": _log(rng, 1, 1000000) - 1, "back": rng.random() < 0.4, "type": s["type"]}
    if kind == "store":
        seqs, heads = _log(rng, 1, 64), s["kv"] * rng.choice((1, 2, 4))
        return {"kind": kind, "seqs": seqs, "rows": _log(rng, 1, max(2, 7500 // seqs)), "len": rng.randrange(0, 600),
                "heads": heads, "turned": rng.choice((0, s["qk"] // 2 * 2, s["qk"] // 4 * 2)), **s}
    if kind == "cross":
        heads = s["kv"] * rng.choice((1, 1, 2, 4))
        rows = rng.choice((1, 4, _log(rng, 5, 500)))
        seqs = _log(rng, 1, 32) if rows < 5 else rng.randrange(1, 5)
        most = min(4000, 65536 // (seqs * s["kv"]) * 8, 60_000_000 // (rows * heads * seqs))
        return {"kind": kind, "seqs": seqs, "rows": rows, "len": _log(rng, 1, max(2, most)), "heads": heads,
                "empty": rng.random() < 0.3, **s}
    heads = s["kv"] * rng.choice((1, 2, 4, 6, 8))
    rows = rng.choice((1, 1, 2, 5, _log(rng, 6, 1000)))
    # keys times rows times heads at most those of a quarter of the largest listed case
    seqs = _log(rng, 1, 64) if rows < 6 else rng.randrange(1, 3)
    most = min(131072 // (seqs * s["kv"]) * 8, 40_000_000 // (rows * heads), 32768)
    span = rng.random() < 0.4
    return {"kind": kind, "seqs": seqs, "rows": rows, "len": rows + _log(rng, 1, max(2, most)), "heads": heads,
            "sink": rng.randrange(0, 130) if span else 0, "ring": _log(rng, 1, 2048) if span else 0, **s}


# ------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1_000_003 + 31)
    return g


def _hip():
    """The framework, imported where its calls are made."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "needle-rs_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import needle_hip
    return needle_hip


def _vectors(g, shape, dtype):
    """Queries, keys or values: channels of different size and offset, as projections give them."""
    d = shape[-1]
    size = torch.exp(0.5 * torch.randn(d, generator=g, device="cuda"))
    offset = 0.5 * torch.randn(d, generator=g, device="cuda")
    return (torch.randn(shape, generator=g, device="cuda") * size + offset).to(TYPES[dtype])


def _lengths(case):
    """The sequences' lengths, the batch's rows among them: the first has the whole of it, the others less."""
    n = case["len"]
    if case["kind"] == "cross":
        out = [max(1, n - (b * 977) % (n // 2 + 1)) for b in range(case["seqs"])]
        return out[:-1] + [0] if case["empty"] else out
    return [max(case["rows"], n - (b * 977) % (n // 2 + 1)) for b in range(case["seqs"])]


def _store_rows(case):
    return [max(1, case["rows"] - (b * 5) % (case["rows"] // 2 + 1)) for b in range(case["seqs"])]


def _cut(case):
    """Positions that a sequence holds before the case's own rows, and those rows, per sequence."""
    if case["kind"] == "store":
        return [case["len"]] * case["seqs"], _store_rows(case)
    lengths = _lengths(case)
    last = [0 if case["kind"] == "cross" else case["rows"]] * case["seqs"]
    return [n - r for n, r in zip(lengths, last)], last


def _inputs(case, seed):
    """What the case's program computed before the call, from the seed alone."""
    g, kind, t = _generator(seed), case["kind"], case["type"]
    if kind == "rope":
        # ragged texts one after the other, each from a position of its own
        n = case["rows"]
        start = torch.randint(0, max(1, n // 3) + 1, (n,), generator=g, device="cuda")
        starts = torch.rand(n, generator=g, device="cuda") < 4.0 / n
        base = torch.cummax(torch.where(starts, torch.arange(n, device="cuda"), 0), 0).values
        positions = case["first"] + torch.arange(n, device="cuda") - base + start[base]
        return {"positions": positions.to(torch.int32), "q": _vectors(g, (n, case["heads"], case["dim"]), t),
                "k": _vectors(g, (n, case["kv"], case["dim"]), t)}
    before, last = _cut(case)
    h, heads, qk, v = case["kv"], case["heads"], case["qk"], case["v"]
    size, offset = (torch.Generator(device="cuda").manual_seed(int(seed) * 7 + i) for i in (1, 2))
    out = {}
    for name, rows in (("0", sum(before)), ("", sum(last))):
        # (the same channels before and after)
        out["k" + name] = _vectors_of(g, size, (rows, h, qk), t)
        out["v" + name] = _vectors_of(g, offset, (rows, h, v), t)
    rows = sum(last) if kind != "cross" else case["seqs"] * case["rows"]
    out["q"] = _vectors(g, (rows, heads, qk), t)
    return out


def _vectors_of(g, channels, shape, dtype):
    """_vectors whose channels' sizes and offsets are another generator's."""
    state = channels.get_state()
    d = shape[-1]
    size = torch.exp(0.5 * torch.randn(d, generator=channels, device="cuda"))
    offset = 0.5 * torch.randn(d, generator=channels, device="cuda")
    channels.set_state(state)
    return (torch.randn(shape, generator=g, device="cuda") * size + offset).to(TYPES[dtype])


# --------------------------------------------------------------- rotations
STRETCH = 8.0       # of the context, where a case scales
ORIGINAL = 8192.0   # positions that the model was made for


def _frequencies(turned, theta, scaling):
    """Radians a position of each pair, in 64 bits, and the amplitude."""
    n = turned // 2
    i = torch.arange(n, dtype=torch.float64)
    if scaling == "base" and turned > 2:
        theta = theta * STRETCH ** (turned / (turned - 2))
    f = theta ** (-2.0 * i / turned)
    if scaling == "linear":
        return f / STRETCH, 1.0
    if scaling == "bands":
        # pairs that turn often within the original length stay, those that turn less than once are stretched
        turns = ORIGINAL * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return f * keep + f / STRETCH * (1.0 - keep), 1.0
    if scaling == "parts":
        # the same between two pairs' indices: 32 turns and 1 turn in the original length
        at = [turned * math.log(ORIGINAL / (r * 2.0 * math.pi)) / (2.0 * math.log(theta)) for r in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), turned - 1)
        keep = 1.0 - ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return f * keep + f / STRETCH * (1.0 - keep), 0.1 * math.log(STRETCH) + 1.0
    return f, 1.0


def _plan(turned, theta, layout, scaling):
    """The framework's plan of the same rotation."""
    nh = _hip()
    args = {"none": None, "linear": ("linear", STRETCH), "base": ("base", STRETCH),
            "bands": ("bands", STRETCH, ORIGINAL), "parts": ("parts", STRETCH, ORIGINAL)}
    return nh.Rope(turned, theta=theta, layout=layout, scaling=args[scaling])


def _turn(x, positions, turned, theta, layout, scaling, back=False):
    """x [rows][heads][dim] turned, in f32; angles in 64 bits."""
    f, amplitude = _frequencies(turned, theta, scaling)
    angle = positions.double()[:, None] * f.to(x.device)
    c = (amplitude * torch.cos(angle)).float()[:, None]
    s = (amplitude * torch.sin(angle)).float()[:, None]
    if back:
        s = -s
    y = x.float().clone()
    n = turned // 2
    a, b = (slice(0, n), slice(n, turned)) if layout == "half" else (slice(0, turned, 2), slice(1, turned, 2))
    xa, xb = x[..., a].float(), x[..., b].float()
    y[..., a] = xa * c - xb * s
    y[..., b] = xb * c + xa * s
    return y


def _store_rope(case):
    return (case["turned"], 10000.0, "half", "none") if case.get("turned") else None


# -------------------------------------------------------------- plain cache
def _pool(case, pages):
    """Empty pages: for keys and for values the numbers [block][head][slot][d] and the steps [block][head]."""
    n = pages * (case["page"] // BLOCK)

    def one(d):
        return [torch.zeros((n, case["kv"], BLOCK, d), dtype=torch.int8, device="cuda"),
                torch.zeros((n, case["kv"]), device="cuda")]
    return one(case["qk"]) + one(case["v"])


def _places(tables, begins, counts, page):
    """Block and slot of positions begins[b] .. + counts[b] of the sequences, by their page lists."""
    at = torch.cat([torch.arange(s, s + n) for s, n in zip(begins, counts)])
    which = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    width = max(1, max(len(t) for t in tables))
    table = torch.tensor([t + [0] * (width - len(t)) for t in tables])
    block = table[which, at // page] * (page // BLOCK) + at % page // BLOCK
    return block.cuda(), (at % BLOCK).cuda()


def _put(codes, steps, x, block, slot):
    """Rows x [row][head][d], f32, into (block[row], slot[row])."""
    if not x.shape[0]:
        return
    touched, of = torch.unique(block, return_inverse=True)
    n, h = touched.numel(), x.shape[1]
    fresh = torch.zeros(n, dtype=torch.bool, device=x.device)
    fresh[of[slot == 0]] = True
    largest = torch.zeros((n, h), device=x.device)
    largest.scatter_reduce_(0, of[:, None].expand(-1, h), x.abs().amax(-1), "amax")
    need = largest / 127.0
    need = torch.where(need < 2.0 ** -120, torch.zeros_like(need), need)
    old = torch.where(fresh[:, None], torch.zeros_like(need), steps[touched])
    k = torch.ceil(torch.log2(need.double() / torch.where(old > 0, old, torch.ones_like(old)).double())).clamp(min=0.0)
    k = torch.where(old > 0, k, torch.zeros_like(k))
    step = torch.where(old > 0, (old.double() * torch.exp2(k)).float(), need)
    steps[touched] = step
    held = codes[touched].float() * torch.exp2(-k).float()[..., None, None]
    codes[touched] = torch.round(held).to(torch.int8)
    inverse = torch.where(step > 0, 1.0 / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(step))
    new = torch.round(x * inverse[of][..., None]).clamp(-127.0, 127.0)
    codes[block, :, slot] = new.to(torch.int8)


def _deal(free, lengths, page):
    """Pages for sequences of these lengths, from the end of the free list."""
    return [[free.pop() for _ in range(-(-n // page))] for n in lengths]


def _shuffled(n, seed):
    return torch.randperm(n, generator=torch.Generator().manual_seed(int(seed) + 5)).tolist()


# ------------------------------------------------------------------ states
def prepare(case, seed):
    """The inputs, and the cache that already holds the sequences' earlier rows."""
    s = {"case": case, **_inputs(case, seed)}
    kind = case["kind"]
    if kind == "rope":
        if own:
            s["rope"] = _plan(case["turned"], case["theta"], case["layout"], case["scaling"])
        return s
    before, last = _cut(case)
    lengths, page = [a + b for a, b in zip(before, last)], case["page"]
    pages = max(1, sum(-(-n // page) for n in lengths))
    rope = _store_rope(case)
    if own:
        nh = _hip()
        cache = nh.KvCache8(1, case["kv"], case["qk"], case["v"], pages=pages, seqs=len(lengths),
                            cap=max(lengths + [1]), page=page)
        seqs = [cache.new_seq() for _ in lengths]
        plan = _plan(*rope) if rope else None
        cache.extend(seqs, before)
        cache.append(0, s["k0"], s["v0"], rope=plan)
        s |= {"cache": cache, "seqs": seqs, "rope": plan, "lengths": lengths, "before": before}
        if kind == "cross":
            cache.ask(seqs, [case["rows"]] * len(seqs))
        else:
            cache.extend(seqs, last)
        if kind == "attend":
            cache.append(0, s["k"], s["v"])
        if kind != "store":
            del s["k"], s["v"]
        del s["k0"], s["v0"]
        return s
    s["pool"] = _pool(case, pages)
    s["tables"] = _deal(_shuffled(pages, seed), lengths, page)
    for name, begins, counts in (("0", [0] * len(before), before), ("", before, last)):
        k, v = s.pop("k" + name), s.pop("v" + name)
        if kind == "store" and not name:
            s |= {"k": k, "v": v, "at": _places(s["tables"], begins, counts, page),
                  "positions": torch.cat([torch.arange(a, a + n) for a, n in zip(begins, counts)]).cuda()}
            continue
        at = _places(s["tables"], begins, counts, page)
        k = k.float()
        if rope and k.shape[0]:
            k = _turn(k, torch.cat([torch.arange(a, a + n) for a, n in zip(begins, counts)]).cuda(), rope[0], rope[1],
                      rope[2], rope[3])
        _put(*s["pool"][:2], k, *at)
        _put(*s["pool"][2:], v.float(), *at)
    if kind == "store":
        first = [a // BLOCK * BLOCK for a in before]
        s["back"] = _places(s["tables"], first, [n - a for n, a in zip(lengths, first)], page)
        return s
    width = max(1, max(len(t) for t in s["tables"]))
    per = page // BLOCK
    table = torch.tensor([t + [0] * (width - len(t)) for t in s["tables"]])
    s["blocks"] = (table[..., None] * per + torch.arange(per)).flatten(1).cuda()
    s["lengths"] = torch.tensor(lengths).cuda()
    return s


# -------------------------------------------------------------------- runs
def _attend_plain(s):
    c = s["case"]
    b, n, h, heads = c["seqs"], c["rows"], c["kv"], c["heads"]

    def held(codes, steps):  # [b][head][position][d]
        x = codes[s["blocks"]].float() * steps[s["blocks"]][..., None, None]
        return x.transpose(1, 2).flatten(2, 3)
    k, v = held(*s["pool"][:2]), held(*s["pool"][2:])
    q = s["q"].float().view(b, n, h, heads // h, c["qk"]).permute(0, 2, 3, 1, 4).reshape(b, h, heads // h * n, c["qk"])
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(c["qk"])
    scores = scores.view(b, h, heads // h, n, -1)
    j = torch.arange(scores.shape[-1], device="cuda")
    if c["kind"] == "cross":
        seen = (j < s["lengths"][:, None])[:, None].expand(-1, n, -1)
    else:
        i = s["lengths"][:, None] - n + torch.arange(n, device="cuda")
        seen = j <= i[..., None]
        if c["ring"]:
            seen = seen & ((j < c["sink"]) | (j > i[..., None] - c["ring"]))
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(most == -math.inf, torch.zeros_like(most), most))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p.view(b, h, heads // h * n, -1), v).view(b, h, heads // h, n, c["v"])
    return o.permute(0, 3, 1, 2, 4).reshape(b * n, heads, c["v"]).to(TYPES[c["type"]])


def run(s):
    """One pass through the operator."""
    c = s["case"]
    kind, t = c["kind"], TYPES[c["type"]]
    if own:
        return _run_own(s, c, kind, t)
    if kind == "rope":
        args = (s["positions"], c["turned"], c["theta"], c["layout"], c["scaling"], c["back"])
        return {"q": _turn(s["q"], *args).to(t), "k": _turn(s["k"], *args).to(t)}
    if kind != "store":
        return _attend_plain(s)
    rope = _store_rope(c)
    k, q = s["k"].float(), None
    if rope:
        k = _turn(k, s["positions"], rope[0], rope[1], rope[2], rope[3])
        q = _turn(s["q"], s["positions"], rope[0], rope[1], rope[2], rope[3]).to(t)
    _put(*s["pool"][:2], k, *s["at"])
    _put(*s["pool"][2:], s["v"].float(), *s["at"])
    block, slot = s["back"]
    out = [(codes[block, :, slot].float() * steps[block][..., None]).to(t) for codes, steps in (s["pool"][:2], s["pool"][2:])]
    return {"q": q, "k": out[0], "v": out[1]} if rope else {"k": out[0], "v": out[1]}


def _run_own(s, c, kind, t):
    if kind == "rope":
        q, k = s["rope"].apply(s["positions"], s["q"], s["k"], transposed=c["back"])
        return {"q": q, "k": k}
    cache = s["cache"]
    if kind != "store":
        return cache.attend(0, s["q"], sink=c.get("sink", 0), ring=c.get("ring", 0))
    first = [a // BLOCK * BLOCK for a in s["before"]]
    if s["rope"] is None:
        cache.append(0, s["k"], s["v"])
    else:
        q = cache.append(0, s["k"], s["v"], rope=s["rope"], q=s["q"])
    k, v = cache.read(0, s["seqs"], first, [n - a for n, a in zip(s["lengths"], first)], t)
    return {"k": k, "v": v} if s["rope"] is None else {"q": q, "k": k, "v": v}


# -------------------------------------------------------------------- work
def _row_bytes(case):
    """A position's numbers and its share of the steps."""
    return case["kv"] * (case["qk"] + case["v"] + 2 * 4 / BLOCK)


def work(case):
    kind, es = case["kind"], 4 if case["type"] == "f32" else 2
    if kind == "rope":
        wide = (case["heads"] + case["kv"]) * case["dim"]
        turned = (case["heads"] + case["kv"]) * case["turned"]
        return {"bytes": case["rows"] * (2 * wide * es + 4), "flops": case["rows"] * 3 * turned}
    wide = case["kv"] * (case["qk"] + case["v"]) * es
    if kind == "store":
        r = sum(_store_rows(case))
        back = r + case["seqs"] * (case["len"] % BLOCK)
        q = 2 * case["heads"] * case["qk"] * es if case["turned"] else 0
        return {"bytes": int(r * (wide + q) + back * (2 * _row_bytes(case) + wide)),
                "flops": (r + back) * 3 * case["kv"] * (case["qk"] + case["v"])}
    n, heads = case["rows"], case["heads"]
    keys = pairs = 0
    for length in _lengths(case):
        if kind == "cross":
            keys += length
            pairs += n * length
        elif case["ring"]:
            first = length - n
            low = max(0, first - case["ring"] + 1)
            keys += length - low + min(case["sink"], low)
            pairs += sum(min(i + 1, min(case["ring"], i + 1) + min(case["sink"], max(0, i + 1 - case["ring"])))
                         for i in range(first, length))
        else:
            keys += length
            pairs += n * length - n * (n - 1) // 2
    io = case["seqs"] * n * heads * (case["qk"] + case["v"]) * es
    return {"bytes": int(keys * _row_bytes(case) + io), "flops": 2 * pairs * heads * (case["qk"] + case["v"])}


# ------------------------------------------------------------------- exact
def _turned64(x, positions, case_rope, back=False):
    """x turned in 64 bits, by complex numbers."""
    turned, theta, layout, scaling = case_rope
    f, amplitude = _frequencies(turned, theta, scaling)
    w = torch.polar(torch.full((), amplitude, dtype=torch.float64, device=x.device),
                    positions.double()[:, None] * f.to(x.device) * (-1.0 if back else 1.0))[:, None]
    x = x.double()
    head, tail = x[..., :turned], x[..., turned:]
    n = turned // 2
    z = head.unflatten(-1, (2, n) if layout == "half" else (n, 2))
    z = z.transpose(-1, -2) if layout == "half" else z
    z = torch.view_as_complex(z.contiguous()) * w
    z = torch.view_as_real(z)
    z = z.transpose(-1, -2) if layout == "half" else z
    return torch.cat((z.flatten(-2), tail), -1)


def _turned32(x, positions, case_rope):
    """Keys as the cache takes them: the format's 32-bit rule, a pair at a time."""
    turned, theta, layout, scaling = case_rope
    f, amplitude = _frequencies(turned, theta, scaling)
    y = x.to(torch.float32).clone()
    n = turned // 2
    for i in range(n):
        a, b = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
        angle = positions.double() * float(f[i])
        c, s = ((amplitude * w(angle)).to(torch.float32)[:, None] for w in (torch.cos, torch.sin))
        xa, xb = x[..., a].to(torch.float32), x[..., b].to(torch.float32)
        y[..., a] = torch.sub(torch.mul(xa, c), torch.mul(xb, s))
        y[..., b] = torch.add(torch.mul(xb, c), torch.mul(xa, s))
    return y


def _held(x, cut):
    """The values that the cache holds for one sequence's rows x [n][head][d], the
    first `cut` of them stored before the others, in 64 bits: steps and whole
    numbers by the format's 32-bit rule, a block at a time."""
    n, h, d = x.shape
    x = x.to(torch.float32)

    def needed(rows):  # [..][row][head][d] -> [..][head]
        m = rows.abs().amax((-3, -1)) / torch.tensor(127.0, device=x.device)
        return m * (m >= 2.0 ** -120)

    def numbers(rows, step):
        r = torch.where(step > 0, torch.reciprocal(step.clamp(min=2.0 ** -121)), torch.zeros_like(step))
        return (rows * r[..., None, :, None]).round().clamp(-127, 127)
    padded = torch.zeros((-(-n // BLOCK) * BLOCK, h, d), device=x.device)
    padded[:n] = x
    whole = padded.unflatten(0, (-1, BLOCK))
    step = needed(whole)
    code = numbers(whole, step)
    b, at = divmod(cut, BLOCK)
    if at and cut < n:
        # the block that was begun before: its step from those rows, doubled as the others need
        old, joined = whole[b, :at], whole[b, at:]
        first, need = needed(old), needed(joined)
        now, shift = first.clone(), torch.zeros_like(first)
        for _ in range(300):
            short = (now > 0) & (now < need)
            if not bool(short.any()):
                break
            now = torch.where(short, now * 2, now)
            shift += short
        now = torch.where(first > 0, now, need)
        before = numbers(old, first).double() * torch.exp2(-shift.double())[:, None]
        step[b] = now
        code[b, :at] = before.round().float()
        code[b, at:] = numbers(joined, now)
    return (code.double() * step.double()[:, None, :, None]).flatten(0, 1)[:n]


def exact(case, seed):
    kind = case["kind"]
    s = _inputs(case, seed)
    if kind == "rope":
        rope = (case["turned"], case["theta"], case["layout"], case["scaling"])
        return {w: _turned64(s[w], s["positions"], rope, case["back"]) for w in ("q", "k")}
    before, last = _cut(case)
    rope = _store_rope(case)
    a0 = a1 = 0
    held = []
    for n0, n1 in zip(before, last):
        k, v = (torch.cat((s[w + "0"][a0:a0 + n0], s[w][a1:a1 + n1])) for w in ("k", "v"))
        if rope and n0 + n1:
            k = _turned32(k, torch.arange(n0 + n1, device="cuda"), rope)
        held.append((_held(k, n0), _held(v, n0)) if n0 + n1 else (k.double(), v.double()))
        a0 += n0
        a1 += n1
    if kind == "store":
        first = [a // BLOCK * BLOCK for a in before]
        out = {w: torch.cat([x[i][a:] for x, a in zip(held, first)]) for i, w in enumerate(("k", "v"))}
        if rope:
            positions = torch.cat([torch.arange(a, a + n) for a, n in zip(before, last)]).cuda()
            out = {"q": _turned64(s["q"], positions, rope), **out}
        return out
    n, per = case["rows"], case["heads"] // case["kv"]
    out = torch.zeros(case["seqs"] * n, case["heads"], case["v"], dtype=torch.float64, device="cuda")
    for b, (k, v) in enumerate(held):
        length = k.shape[0]
        if not length:
            continue
        i = torch.arange(length - n, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")
        hidden = j > i if kind == "attend" else torch.zeros((n, length), dtype=torch.bool, device="cuda")
        if case.get("ring"):
            hidden = hidden | ((j >= case["sink"]) & (j <= i - case["ring"]))
        for head in range(case["heads"]):
            q = s["q"][b * n:(b + 1) * n, head].double()
            z = q @ k[:, head // per].t().contiguous() * (1.0 / math.sqrt(case["qk"]))
            z[hidden] = -math.inf
            out[b * n:(b + 1) * n, head] = torch.softmax(z, -1) @ v[:, head // per].contiguous()
    return out
