"""The operators of a 4-bit key/value cache and of drafted decoding, as measurable cases.

Each case can be run in two forms on the same inputs: with ``own`` false the
operator written out in elementary torch operations, with ``own`` true the
framework's calls (`needle_hip.KvCache4`, `needle_hip.verify_drafts`).

The cache holds rows of keys and values in groups of 32 or 64 along the head:
low = f16(min), step = f16((max - min) * f32(1/15)), code = round((x - low) *
(1 / step)) in 0..15, all in f32; the value held is low + step * code.

Kinds:
  store    new rows of every sequence of a batch into the cache, and the values held in their place
  fork     branches of one prefix: pages shared, the last one copied on write, a few rows of their own
           in every layer, the branches' contents read, the branches freed
  copy     a sequence's pages copied into pages of its own, its contents read
  compact  branches of sequences that keep some ranges of positions, closed up, their contents read
  attend   attention of each sequence's last rows over its 4-bit cache, with first positions that stay
           visible (sink) and a window of last ones (ring; 0: all)
  verify   drafted tokens against the target's logits and given random numbers
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    agent = {"kv": 2, "qk": 48, "v": 64, "group": 32, "page": 32, "type": "f32"}
    wide = {"kv": 8, "qk": 128, "v": 128, "group": 32, "page": 64}
    return [
        # One decoding step of eight conversations: a layer's new rows, at the
        # published model's head shapes. Launches and host time count.
        {"name": "store_step", "kind": "store", "seqs": 8, "rows": 1, "len": 300, **agent},
        # Prompts of several requests into one layer of a wider model.
        {"name": "store_prompts", "kind": "store", "seqs": 3, "rows": 2500, "len": 77, **wide, "type": "bf16"},
        # The agent's static prefix, branched for eight candidate continuations.
        {"name": "fork_prefix", "kind": "fork", "layers": 20, "len": 118, "branches": 8, "rows": 3, **agent},
        # Long conversations cut back to their prefix and the last positions.
        {"name": "compact_span", "kind": "compact", "layers": 8, "seqs": 3, "len": 4000, "kept": 1374, "pieces": 2,
         **wide, "type": "bf16"},
        # A decoding step of one agent turn under its span of 118 + 256 positions.
        {"name": "step_agent", "kind": "attend", "seqs": 1, "rows": 1, "len": 700, "heads": 12, "sink": 118, "ring": 256,
         **agent},
        # A server's decoding step: 64 conversations of up to 8192 positions.
        {"name": "step_batch", "kind": "attend", "seqs": 64, "rows": 1, "len": 8192, "heads": 32, "sink": 0, "ring": 0,
         **wide, "type": "bf16"},
        # One conversation over a very long document, larger groups.
        {"name": "step_document", "kind": "attend", "seqs": 1, "rows": 1, "len": 131072, "heads": 32, "sink": 0,
         "ring": 0, **wide, "group": 64, "type": "f16"},
        # The check of four drafted tokens in 16 conversations, windowed layers.
        {"name": "drafts_window", "kind": "attend", "seqs": 16, "rows": 5, "len": 5000, "heads": 32, "sink": 4,
         "ring": 1024, **wide, "type": "bf16"},
        # A chunk of two long prompts: the queries of 2000 positions after 6000.
        {"name": "prompt_chunk", "kind": "attend", "seqs": 2, "rows": 2000, "len": 8000, "heads": 32, "sink": 0,
         "ring": 0, **wide, "type": "bf16"},
        # Four drafted tokens of one agent turn, looked up in its prompt (no
        # probabilities of their own), at the published vocabulary.
        {"name": "verify_agent", "kind": "verify", "seqs": 1, "drafts": 4, "vocab": 8192, "type": "f32", "probs": False,
         "temperature": 0.7},
        # The same for eight conversations decoding greedily over the benchmark's head.
        {"name": "verify_greedy", "kind": "verify", "seqs": 8, "drafts": 7, "vocab": 32768, "type": "f32",
         "probs": False, "temperature": 0.0},
        # A server's step with a draft model: 32 conversations, five drafts each.
        {"name": "verify_batch", "kind": "verify", "seqs": 32, "drafts": 5, "vocab": 131072, "type": "bf16",
         "probs": True, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _shape(rng):
    """Heads, head widths, group, page and type of a drawn case."""
    qk, v = rng.choice(((48, 64), (64, 64), (80, 80), (96, 96), (128, 128), (128, 128), (192, 128), (256, 256), (45, 51)))
    return {"kv": rng.choice((1, 2, 3, 4, 8)), "qk": qk, "v": v, "group": rng.choice((32, 64)),
            "page": rng.choice((32, 64, 128)), "type": rng.choice(("f32", "bf16", "bf16", "f16"))}


def draw(rng):
    """One more case of the listed ones' ranges."""
    kind = rng.choice(("store", "fork", "copy", "compact", "attend", "attend", "attend", "attend", "verify", "verify"))
    s = _shape(rng)
    if kind == "store":
        seqs = _log(rng, 1, 64)
        return {"kind": kind, "seqs": seqs, "rows": _log(rng, 1, max(2, 7500 // seqs)), "len": rng.randrange(0, 2000), **s}
    if kind == "fork":
        return {"kind": kind, "layers": rng.randrange(1, 21), "len": rng.randrange(1, 400),
                "branches": rng.randrange(1, 9), "rows": rng.randrange(1, 6), **s, "kv": min(s["kv"], 2)}
    if kind == "copy":
        return {"kind": kind, "layers": rng.randrange(1, 9), "len": _log(rng, 1, 4000), **s}
    if kind == "compact":
        length = _log(rng, 40, 4000)
        kept = rng.randrange(1, length // 2 + 1)
        return {"kind": kind, "layers": rng.randrange(1, 9), "seqs": rng.randrange(1, 4), "len": length, "kept": kept,
                "pieces": rng.randrange(1, min(kept, 40) + 1), **s}
    if kind == "attend":
        heads = s["kv"] * rng.choice((1, 2, 4, 6, 8))
        rows = rng.choice((1, 1, 2, 5, _log(rng, 6, 1000)))
        # keys times rows times heads at most those of a quarter of the largest listed case
        seqs = _log(rng, 1, 64) if rows < 6 else rng.randrange(1, 3)
        most = min(131072 // (seqs * s["kv"]) * 8, 40_000_000 // (rows * heads), 32768)
        length = rows + _log(rng, 1, max(2, most))
        span = rng.random() < 0.4
        return {"kind": kind, "seqs": seqs, "rows": rows, "len": length, "heads": heads,
                "sink": rng.randrange(0, 130) if span else 0, "ring": _log(rng, 1, 2048) if span else 0, **s}
    vocab = _log(rng, 500, 131072)
    drafts = rng.randrange(0, 9)
    return {"kind": kind, "seqs": _log(rng, 1, max(2, min(64, 32 * 6 * 131072 // (vocab * (drafts + 1))))),
            "drafts": drafts, "vocab": vocab, "type": s["type"], "probs": rng.random() < 0.5,
            "temperature": rng.choice((0.0, 0.6, 1.0, 1.3))}


# ------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1_000_003 + 29)
    return g


def _hip():
    """The framework, imported where its calls are made."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "needle-rs_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import needle_hip
    return needle_hip


def _vectors(g, shape, dtype):
    """Keys or values: channels of different size and offset, as projections give them."""
    d = shape[-1]
    size = torch.exp(0.5 * torch.randn(d, generator=g, device="cuda"))
    offset = 0.5 * torch.randn(d, generator=g, device="cuda")
    return (torch.randn(shape, generator=g, device="cuda") * size + offset).to(TYPES[dtype])


def _lengths(case):
    """The sequences' lengths, the last rows among them: the first has the whole of it, the others less."""
    n, rows = case["len"], case["rows"]
    return [max(rows, n - (b * 977) % (n // 2 + 1)) for b in range(case["seqs"])]


def _store_rows(case):
    return [max(1, case["rows"] - (b * 5) % (case["rows"] // 2 + 1)) for b in range(case["seqs"])]


def _pieces(case, b):
    """The ranges of positions that sequence b keeps: ascending, apart, the last one at its end."""
    n, kept, pieces = case["len"], case["kept"], case["pieces"]
    gaps = n - kept
    ranges, at = [], 0
    for i in range(pieces):
        size = kept * (i + 1) // pieces - kept * i // pieces
        ranges.append((at, at + size))
        at += size + (gaps * (i + 1) // max(1, pieces - 1) - gaps * i // max(1, pieces - 1) if pieces > 1 else 0)
    if pieces == 1:
        ranges = [(gaps, n)]
    shift = b % 3 if ranges[-1][1] - ranges[-1][0] > 3 else 0
    return ranges[:-1] + [(ranges[-1][0] + shift, ranges[-1][1])]


def _inputs(case, seed):
    """What the case's program computed before the call, from the seed alone."""
    g, kind, t = _generator(seed), case["kind"], case["type"]
    if kind == "verify":
        b, n, v = case["seqs"], case["drafts"], case["vocab"]
        logits = 2.5 * torch.randn(b, n + 1, v, generator=g, device="cuda")
        logits += 3.0 * (torch.rand(b, n + 1, v, generator=g, device="cuda") < 20.0 / v)
        draft = torch.softmax(logits[:, :n] + 0.6 * torch.randn(b, n, v, generator=g, device="cuda"), -1)
        x = torch.zeros(b, n, dtype=torch.int64, device="cuda")
        if n:
            x = torch.multinomial(draft.reshape(b * n, v), 1, generator=g).view(b, n)
        if case["temperature"] == 0.0 or not case["probs"]:
            # a drafter that is mostly right: the likeliest token, or any
            best = logits[:, :n].argmax(-1)
            x = torch.where(torch.rand(b, n, generator=g, device="cuda") < 0.8, best, x)
        u = torch.rand(b, n + 1, generator=g, device="cuda")
        return {"logits": logits.to(TYPES[t]), "drafts": x.to(torch.int32), "u": u,
                "probs": draft if case["probs"] else None}
    h, qk, v = case["kv"], case["qk"], case["v"]
    if kind == "store":
        r = sum(_store_rows(case))
        return {"k": _vectors(g, (r, h, qk), t), "v": _vectors(g, (r, h, v), t)}
    if kind == "attend":
        r = sum(_lengths(case))
        q = _vectors(g, (case["seqs"] * case["rows"], case["heads"], qk), t)
        return {"q": q, "k": _vectors(g, (r, h, qk), t), "v": _vectors(g, (r, h, v), t)}
    r = case["len"] * case.get("seqs", 1)
    out = {"k": _vectors(g, (case["layers"], r, h, qk), t), "v": _vectors(g, (case["layers"], r, h, v), t)}
    if kind == "fork":
        m = case["branches"] * case["rows"]
        out |= {"k2": _vectors(g, (case["layers"], m, h, qk), t), "v2": _vectors(g, (case["layers"], m, h, v), t)}
    return out


# -------------------------------------------------------------- plain cache
def _pack(x, group):
    """Rows [..., d] as two codes a byte, and the groups' steps and lows in f16."""
    d = x.shape[-1]
    n = -(-d // group)
    x = x.float().clamp(-65504.0, 65504.0)
    at = (torch.arange(n * group, device=x.device)).clamp(max=d - 1)
    parts = x[..., at].unflatten(-1, (n, group))
    least, most = parts.amin(-1), parts.amax(-1)
    low = least.half()
    step = ((most - least) * torch.tensor(1.0 / 15.0, device=x.device)).half()
    inverse = 1.0 / torch.where(step > 0, step.float(), torch.ones_like(least))
    codes = torch.round((parts - low.float()[..., None]) * inverse[..., None]).clamp(0, 15)
    codes = torch.where(step[..., None] > 0, codes, torch.zeros_like(codes)).to(torch.uint8).flatten(-2)[..., :d]
    if d % 2:
        codes = torch.nn.functional.pad(codes, (0, 1))
    return codes[..., 0::2] | (codes[..., 1::2] << 4), step, low


def _unpack(codes, step, low, d, group):
    """The values held, in f32."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :d].float()
    at = torch.arange(d, device=codes.device) // group
    return low.float()[..., at] + step.float()[..., at] * c


def _pool(case, layers, pages):
    """Empty pages: for keys and for values the codes, steps and lows, [page][layer][head][slot][..]."""
    h, page, group = case["kv"], case["page"], case["group"]

    def one(d):
        n = -(-d // group)
        return [torch.zeros((pages, layers, h, page, w), dtype=t, device="cuda")
                for w, t in ((-(-d // 2), torch.uint8), (n, torch.float16), (n, torch.float16))]
    return one(case["qk"]) + one(case["v"])


def _put(pool, case, pages, slots, k, v):
    """Rows k, v [layer][row][head][d] into (pages[row], slots[row])."""
    for part, x in zip(pool, _pack(k, case["group"]) + _pack(v, case["group"])):
        part[pages, :, :, slots] = x.transpose(0, 1)


def _get(pool, case, pages, slots):
    """The values held at (pages[row], slots[row]): k, v [layer][row][head][d] in the case's type."""
    parts = [p[pages, :, :, slots].transpose(0, 1) for p in pool]
    k = _unpack(*parts[:3], case["qk"], case["group"])
    v = _unpack(*parts[3:], case["v"], case["group"])
    return k.to(TYPES[case["type"]]), v.to(TYPES[case["type"]])


def _places(tables, begins, counts, page):
    """Page and slot of positions begins[b] .. + counts[b] of the sequences, by their page lists."""
    at = torch.cat([torch.arange(s, s + n) for s, n in zip(begins, counts)])
    which = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    width = max(len(t) for t in tables)
    table = torch.tensor([t + [0] * (width - len(t)) for t in tables])
    return table[which, at // page].cuda(), (at % page).cuda()


def _deal(free, lengths, page):
    """Pages for sequences of these lengths, from the end of the free list."""
    return [[free.pop() for _ in range(-(-n // page))] for n in lengths]


def _shuffled(n, seed):
    return torch.randperm(n, generator=torch.Generator().manual_seed(int(seed) + 5)).tolist()


# ------------------------------------------------------------------ states
def _cache_lengths(case):
    kind = case["kind"]
    if kind == "store":
        return [case["len"] + r for r in _store_rows(case)]
    if kind == "attend":
        return _lengths(case)
    return [case["len"]] * case.get("seqs", 1)


def prepare(case, seed):
    """The inputs, and the cache that already holds the sequences' earlier rows."""
    s = {"case": case, **_inputs(case, seed)}
    kind = case["kind"]
    if kind == "verify":
        return s
    lengths, page, layers = _cache_lengths(case), case["page"], case.get("layers", 1)
    pages = sum(-(-n // page) for n in lengths)
    extra = {"fork": case.get("branches", 0) * (-(-case.get("rows", 0) // page) + 1), "copy": pages,
             "compact": pages + len(lengths)}.get(kind, 0)
    if own:
        nh = _hip()
        width = max(-(-n // page) for n in lengths) * page + page
        cache = nh.KvCache4(layers, case["kv"], case["qk"], case["v"], pages=pages + extra,
                            seqs=len(lengths) * 2 + case.get("branches", 0), cap=width, group=case["group"], page=page)
        seqs = [cache.new_seq() for _ in lengths]
        last = {"store": _store_rows, "attend": lambda c: [c["rows"]] * c["seqs"]}.get(kind, lambda c: [0] * len(seqs))(case)
        before = [n - r for n, r in zip(lengths, last)]
        s |= {"cache": cache, "seqs": seqs, "before": before, "last": last}
        cache.extend(seqs, before)
        if kind == "store":
            cache.extend(seqs, last)
        elif kind == "attend":
            # earlier rows first, then the batch's own, as its program wrote them
            ends = torch.tensor(lengths).cumsum(0)
            own_rows = torch.cat([torch.arange(e - case["rows"], e) for e in ends.tolist()]).cuda()
            keep = torch.ones(s["k"].shape[0], dtype=torch.bool, device="cuda")
            keep[own_rows] = False
            cache.append(0, s["k"][keep], s["v"][keep])
            cache.extend(seqs, last)
            cache.append(0, s["k"][own_rows], s["v"][own_rows])
            del s["k"], s["v"]
        else:
            for layer in range(layers):
                cache.append(layer, s["k"][layer], s["v"][layer])
            del s["k"], s["v"]
        return s
    free = _shuffled(pages + extra, seed)
    s["pool"] = _pool(case, layers, pages + extra)
    s["tables"] = _deal(free, lengths, page)
    s["free"] = free
    if kind == "store":
        rows = _store_rows(case)
        s["at"] = _places(s["tables"], [case["len"]] * len(rows), rows, page)
        return s
    k, v = s.pop("k"), s.pop("v")
    if kind == "attend":
        k, v = k[None], v[None]
        width = max(len(t) for t in s["tables"])
        s["table"] = torch.tensor([t + [0] * (width - len(t)) for t in s["tables"]]).cuda()
        s["lengths"] = torch.tensor(lengths).cuda()
    _put(s["pool"], case, *_places(s["tables"], [0] * len(lengths), lengths, page), k, v)
    return s


# -------------------------------------------------------------------- runs
def _attend_plain(s):
    c = s["case"]
    b, n, h, heads = c["seqs"], c["rows"], c["kv"], c["heads"]
    held = [p[s["table"], 0].transpose(1, 2).flatten(2, 3) for p in s["pool"]]  # [b][head][position][..]
    k = _unpack(*held[:3], c["qk"], c["group"])
    v = _unpack(*held[3:], c["v"], c["group"])
    q = s["q"].float().view(b, n, h, heads // h, c["qk"]).permute(0, 2, 3, 1, 4).reshape(b, h, heads // h * n, c["qk"])
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(c["qk"])
    scores = scores.view(b, h, heads // h, n, -1)
    j = torch.arange(scores.shape[-1], device="cuda")
    i = s["lengths"][:, None] - n + torch.arange(n, device="cuda")
    seen = j <= i[..., None]
    if c["ring"]:
        seen &= (j < c["sink"]) | (j > i[..., None] - c["ring"])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, h, heads // h * n, -1), v).view(b, h, heads // h, n, c["v"])
    return o.permute(0, 3, 1, 2, 4).reshape(b * n, heads, c["v"]).to(TYPES[c["type"]])


def _verify_plain(s):
    """In 64 bits: sums over the vocabulary, and picks next to a border."""
    c = s["case"]
    b, n, vocab, t = c["seqs"], c["drafts"], c["vocab"], c["temperature"]
    x, u = s["drafts"].long(), s["u"].double()
    each = torch.arange(b, device="cuda")
    if t == 0.0:
        best = s["logits"].float().argmax(-1)
        good = x == best[:, :n]
    else:
        logits = s["logits"].double()
        p = torch.exp((logits - logits.amax(-1, keepdim=True)) / t)
        p = p / p.sum(-1, keepdim=True)
        px = p[:, :n].gather(-1, x[..., None])[..., 0]
        qx = s["probs"].double().gather(-1, x[..., None])[..., 0] if c["probs"] else torch.ones_like(px)
        good = u[:, :n] * qx < px
    accepted = torch.cumprod(good.long(), -1).sum(-1)
    if t == 0.0:
        pick = best[each, accepted]
    else:
        w = p[each, accepted]
        refused = accepted < n
        if n:
            at = accepted.clamp(max=n - 1)
            if c["probs"]:
                rest = (w - s["probs"][each, at].double()).clamp(min=0)
            else:
                rest = w.scatter(-1, x[each, at][:, None], 0.0)
            rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
            w = torch.where(refused[:, None], rest, w)
        total = torch.cumsum(w, -1)
        pick = (total <= u[:, n:] * total[:, -1:]).sum(-1)
        last = vocab - 1 - (w > 0).flip(-1).long().argmax(-1)
        pick = torch.minimum(pick, last)
    at = torch.arange(n + 1, device="cuda")
    drafts = torch.cat((x, x.new_zeros(b, 1)), -1)
    tokens = torch.where(at < accepted[:, None], drafts, torch.where(at == accepted[:, None], pick[:, None], -1))
    return {"accepted": accepted.to(torch.int32), "tokens": tokens.to(torch.int32)}


def run(s):
    """One pass through the operator."""
    c = s["case"]
    kind = c["kind"]
    if own:
        return _run_own(s, c, kind)
    page = c["page"] if kind != "verify" else 0
    if kind == "verify":
        return _verify_plain(s)
    if kind == "attend":
        return _attend_plain(s)
    pool = s["pool"]
    if kind == "store":
        _put(pool, c, *s["at"], s["k"][None], s["v"][None])
        k, v = _get(pool, c, *s["at"])
        return {"k": k[0], "v": v[0]}
    free = list(s["free"])
    if kind == "fork":
        n, m, whole = c["len"], c["branches"], c["len"] // page
        first = s["tables"][0]
        tables = [first[:whole] + [free.pop() for _ in range(-(-(n + c["rows"]) // page) - whole)] for _ in range(m)]
        if n % page:
            copied = torch.tensor([t[whole] for t in tables]).cuda()
            for part in pool:
                part[copied] = part[first[whole]].clone()
        _put(pool, c, *_places(tables, [n] * m, [c["rows"]] * m, page), s["k2"], s["v2"])
        k, v = _get(pool, c, *_places(tables, [0] * m, [n + c["rows"]] * m, page))
        return {"k": k, "v": v}
    if kind == "copy":
        table = [free.pop() for _ in s["tables"][0]]
        source, target = torch.tensor(s["tables"][0]).cuda(), torch.tensor(table).cuda()
        for part in pool:
            part[target] = part[source]
        k, v = _get(pool, c, *_places([table], [0], [c["len"]], page))
        return {"k": k, "v": v}
    ranges = [_pieces(c, b) for b in range(c["seqs"])]
    kept = [sum(e - a for a, e in r) for r in ranges]
    tables = _deal(free, kept, page)
    pages, slots = _places([t for t, r in zip(s["tables"], ranges) for _ in r], [a for r in ranges for a, _ in r],
                           [e - a for r in ranges for a, e in r], page)
    to = _places(tables, [0] * len(kept), kept, page)
    for part in pool:
        part[to[0], :, :, to[1]] = part[pages, :, :, slots]
    k, v = _get(pool, c, *to)
    return {"k": k, "v": v}


def _run_own(s, c, kind):
    if kind == "verify":
        accepted, tokens = _hip().verify_drafts(s["logits"], s["drafts"], s["u"], probs=s["probs"],
                                                temperature=c["temperature"])
        return {"accepted": accepted, "tokens": tokens}
    cache, seqs, t = s["cache"], s["seqs"], TYPES[c["type"]]
    if kind == "attend":
        return cache.attend(0, s["q"], scale=1.0 / math.sqrt(c["qk"]), sink=c["sink"], ring=c["ring"])
    if kind == "store":
        cache.append(0, s["k"], s["v"])
        k, v = cache.read(0, seqs, s["before"], s["last"], t)
        return {"k": k, "v": v}
    if kind == "fork":
        made = cache.fork(seqs[0], c["branches"])
        cache.extend(made, [c["rows"]] * len(made))
        for layer in range(c["layers"]):
            cache.append(layer, s["k2"][layer], s["v2"][layer])
        lengths = [c["len"] + c["rows"]] * len(made)
    elif kind == "copy":
        made, lengths = [cache.copy(seqs[0])], [c["len"]]
    else:
        made = [cache.fork(q, 1)[0] for q in seqs]
        ranges = [_pieces(c, b) for b in range(c["seqs"])]
        cache.compact(made, ranges)
        lengths = [sum(e - a for a, e in r) for r in ranges]
    k, v = cache.read(None, made, [0] * len(made), lengths, t)
    for q in made:
        cache.free(q)
    return {"k": k, "v": v}


# -------------------------------------------------------------------- work
def _row_bytes(case):
    """A row's codes, steps and lows in one layer."""
    sides = [(-(-d // 2) + 4 * -(-d // case["group"])) for d in (case["qk"], case["v"])]
    return case["kv"] * sum(sides)


def work(case):
    kind, es = case["kind"], 4 if case["type"] == "f32" else 2
    if kind == "verify":
        rows = case["seqs"] * (case["drafts"] + 1)
        return {"bytes": rows * (case["vocab"] * es + 12), "flops": 3 * rows * case["vocab"]}
    wide = case["kv"] * (case["qk"] + case["v"]) * es
    held = _row_bytes(case)
    if kind == "store":
        r = sum(_store_rows(case))
        return {"bytes": r * (2 * wide + 2 * held), "flops": r * 6 * case["kv"] * (case["qk"] + case["v"])}
    if kind == "attend":
        n, heads = case["rows"], case["heads"]
        keys = pairs = 0
        for length in _lengths(case):
            if case["ring"]:
                first = length - n
                low = max(0, first - case["ring"] + 1)
                keys += length - low + min(case["sink"], low)
                pairs += sum(min(i + 1, min(case["ring"], i + 1) + min(case["sink"], max(0, i + 1 - case["ring"])))
                             for i in range(first, length))
            else:
                keys += length
                pairs += n * length - n * (n - 1) // 2
        io = case["seqs"] * n * heads * (case["qk"] + case["v"]) * es
        return {"bytes": keys * held + io, "flops": 2 * pairs * heads * (case["qk"] + case["v"])}
    layers, length = case["layers"], case["len"]
    if kind == "fork":
        tail = length % case["page"]
        new, whole = case["branches"] * case["rows"], case["branches"] * (length + case["rows"])
        moved = (new + case["branches"] * tail + tail + length) * held + (new + whole) * wide
        return {"bytes": layers * moved, "flops": layers * 2 * whole * case["kv"] * (case["qk"] + case["v"])}
    rows = length if kind == "copy" else case["seqs"] * case["kept"]
    return {"bytes": layers * rows * (3 * held + wide), "flops": layers * 2 * rows * case["kv"] * (case["qk"] + case["v"])}


# ------------------------------------------------------------------- exact
def _held(x, group):
    """The values that the cache holds for rows x, in 64 bits: codes by the
    format's 32-bit rule, a group at a time."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    third = torch.full((), 1.0 / 15.0, dtype=torch.float32, device=x.device)
    for at in range(0, x.shape[-1], group):
        y = x[..., at:at + group].to(torch.float32)
        y = torch.minimum(torch.maximum(y, y.new_tensor(-65504.0)), y.new_tensor(65504.0))
        a, z = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        low, step = a.to(torch.float16), ((z - a) * third).to(torch.float16)
        c = torch.round((y - low.float()) * (1.0 / step.float())).clamp(0.0, 15.0)
        c[(step <= 0).expand_as(c)] = 0.0
        out[..., at:at + group] = low.double() + step.double() * c.double()
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "verify":
        return None
    s = _inputs(case, seed)
    group = case["group"]
    if kind == "store":
        return {"k": _held(s["k"], group), "v": _held(s["v"], group)}
    if kind == "attend":
        n, per = case["rows"], case["heads"] // case["kv"]
        out = torch.empty(case["seqs"] * n, case["heads"], case["v"], dtype=torch.float64, device="cuda")
        at = 0
        for b, length in enumerate(_lengths(case)):
            k, v = (_held(s[w][at:at + length], group) for w in ("k", "v"))
            at += length
            i = torch.arange(length - n, length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")
            hidden = j > i
            if case["ring"]:
                hidden = hidden | ((j >= case["sink"]) & (j <= i - case["ring"]))
            for head in range(case["heads"]):
                q = s["q"][b * n:(b + 1) * n, head].double()
                z = q @ k[:, head // per].t().contiguous() * (1.0 / math.sqrt(case["qk"]))
                z[hidden] = -math.inf
                out[b * n:(b + 1) * n, head] = torch.softmax(z, -1) @ v[:, head // per].contiguous()
        return out
    n = case["len"]
    k, v = _held(s["k"], group), _held(s["v"], group)
    if kind == "copy":
        return {"k": k, "v": v}
    if kind == "fork":
        r = case["rows"]
        k2, v2 = _held(s["k2"], group), _held(s["v2"], group)
        join = lambda x, y: torch.cat([z for m in range(case["branches"]) for z in (x, y[:, m * r:(m + 1) * r])], 1)  # noqa: E731
        return {"k": join(k, k2), "v": join(v, v2)}
    rows = [b * n + i for b in range(case["seqs"]) for a, e in _pieces(case, b) for i in range(a, e)]
    return {"k": k[:, rows], "v": v[:, rows]}
