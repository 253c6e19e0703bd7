"""What a transformer block on int8 products needs around them, as timed cases: the RMS norm whose output is the next
product's 8-bit operand, the key/value cache that is quantised as it is written and read back, and the attention over it.

``own`` false: the plain forms, in torch operations.  ``own`` true: the calls of nnops_b200.ops.

The cache: codes s8 [pages, heads, page tokens, dim] and one f32 scale for each page and head, for keys and for values.  Token t
of sequence b lies in page ``page_table[b, t // page tokens]``.  ``lens[b]`` counts the tokens of a sequence with the new ones;
rows ``cu[b] .. cu[b + 1]`` of the new tokens (or queries) are its last ones.
"""
import math
import random

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-6
_LEAST = 2.0 ** -60    # of a cache's scale


def _norm(name, rows, cols, x, residual):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "x": x, "residual": residual}


def _cache(name, op, seqs, new, length, heads, dim, page, x, ragged):
    return {"name": name, "op": op, "seqs": seqs, "new": new, "len": length, "heads": heads, "dim": dim, "page": page, "x": x,
            "ragged": ragged}


def _attention(name, seqs, new, length, heads, group, dim, page, x, ragged, window=0, sinks=0):
    return _cache(name, "attention", seqs, new, length, heads, dim, page, x, ragged) | {"group": group, "window": window, "sinks": sinks}


def listed():
    return [
        # One token of one user, between two layers.
        _norm("norm_1row", 1, 4096, "f16", True),
        # A prompt between two layers.
        _norm("norm_prompt", 4096, 8192, "f16", True),
        # A small model's rows, off every multiple of a vector, where the residual is added elsewhere.
        _norm("norm_ragged", 333, 1000, "f32", False),
        # A serving batch appends a token to each sequence: nearly always inside a page that is in use.
        _cache("write_decode", "write", 64, 1, 8192, 8, 128, 64, "f16", True),
        # Prompts of several users come in at once, some of them behind a prefix that is there.
        _cache("write_prompts", "write", 8, 2048, 4096, 8, 128, 16, "bf16", True),
        # Contexts are read back, for a layer that wants them as floats.
        _cache("read_contexts", "read", 16, 4096, 4096, 8, 128, 128, "f16", False),
        # The same from a small cache of odd sizes.
        _cache("read_odd", "read", 5, 777, 1500, 5, 96, 32, "f32", True),
        # One user's next token: latency.
        _attention("decode_1seq", 1, 1, 4096, 8, 4, 128, 64, "f16", False),
        # The next token of a serving batch, some of its slots nearly new, one empty.
        _attention("decode_batch", 64, 1, 8192, 8, 8, 128, 64, "bf16", True),
        # Five proposed tokens a sequence are verified at once, behind a sliding window with its first tokens kept.
        _attention("verify_window", 16, 5, 32768, 8, 4, 64, 16, "f16", True, 4096, 4),
        # A long prompt attends to itself.
        _attention("prefill_prompt", 1, 8192, 8192, 8, 4, 128, 128, "f16", False),
        # Chunks of several prompts over what is there of them already.
        _attention("prefill_chunks", 8, 512, 16384, 4, 8, 128, 32, "bf16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        for k, v in work(c).items():
            most[c["op"], k] = max(most.get((c["op"], k), 0), v)
    while True:
        op = rng.choice(["norm", "write", "read", "attention", "attention", "attention"])
        x = rng.choice(["f16", "f16", "bf16", "f32"])
        if op == "norm":
            c = _norm("", _log(rng, 1, 8192), _log(rng, 64, 16384), x, rng.random() < 0.7)
        else:
            heads, dim, page = _log(rng, 1, 16), rng.choice([64, 96, 128, 128, 256]), rng.choice([16, 32, 64, 128])
            seqs, length = _log(rng, 1, 64), _log(rng, 1, 32768)
            ragged = rng.random() < 0.6
            if op == "attention":
                decode = rng.random() < 0.6
                new = _log(rng, 1, 8) if decode else _log(rng, 8, 8192)
                if not decode:
                    x = rng.choice(["f16", "bf16"])    # what prompts are computed in
                window = _log(rng, 16, 8192) if rng.random() < 0.3 else 0
                c = _attention("", seqs, new, length, heads, rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 16]), dim, page, x, ragged, window,
                               rng.randint(0, 8) if window else 0)
            else:
                c = _cache("", op, seqs, 1 if rng.random() < 0.3 else _log(rng, 1, 8192), length, heads, dim, page, x, ragged)
            c["new"] = min(c["new"], c["len"])
        if all(v <= most[op, k] for k, v in work(c).items()) and _room(c) <= 12e9:
            del c["name"]
            return c


def _room(c):
    """Bytes of the largest tensors of the plain form."""
    if c["op"] == "norm":
        return 0
    pages = -(-c["len"] // c["page"]) * c["page"] * c["seqs"]
    kv = 8 * pages * c["heads"] * c["dim"]
    return kv if c["op"] != "attention" else max(kv, 4 * pages * c["new"] * c["heads"] * c["group"])


def _sequences(c):
    """(tokens with the new ones, new ones) of each sequence, in ascending order of their lengths."""
    n, top, new = c["seqs"], c["len"], c["new"]
    if not c["ragged"]:
        return [(top, new)] * n
    both = []
    for i in range(n):
        length = max(1, round(top * (i + 1) / n))
        fresh = new if new == 1 else max(1, round(new * (n - i) / n))
        both.append((length, min(length, fresh)))
    if n >= 8:
        both[0] = (0, 1 if new == 1 else 0)    # a slot of the batch that holds nothing
    return both


def _visible(c):
    """Pairs of query and key that see each other, and keys of every sequence that some query sees."""
    pairs = keys = 0
    for length, new in _sequences(c):
        first, window, sinks = length - new, c["window"], c["sinks"]
        for p in range(max(0, first), length) if window else ():
            pairs += min(p + 1, window + min(sinks, max(0, p + 1 - window)))
        if not window:
            pairs += (length * (length + 1) - max(0, first) * (max(0, first) + 1)) // 2
            keys += length
        else:
            low = max(0, first - window + 1)
            keys += length - low + min(sinks, low)
    return pairs, keys


def work(c):
    b = _BYTES[c["x"]]
    if c["op"] == "norm":
        cells = c["rows"] * c["cols"]
        # x, residual, their sum, the codes' values, weights and scales.
        values = 2 if c["x"] == "f16" else 4
        return {"bytes": cells * (b * (3 if c["residual"] else 1) + values) + c["cols"] * b + 4 * c["rows"], "flops": 6 * cells}
    row = c["heads"] * c["dim"]
    fresh = sum(new for length, new in _sequences(c) if length)
    if c["op"] == "write":
        return {"bytes": 2 * row * fresh * (b + 1 + b), "flops": 8 * row * fresh}
    if c["op"] == "read":
        return {"bytes": 2 * row * fresh * (1 + b), "flops": 2 * row * fresh}
    pairs, keys = _visible(c)
    rows = sum(new for _, new in _sequences(c))
    return {"bytes": 2 * row * keys + 8 * c["heads"] * keys / c["page"] + 2 * b * rows * row * c["group"],
            "flops": 4 * pairs * row * c["group"]}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _generator(seed)
    x = _TYPES[case["x"]]
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "norm":
        m, n = case["rows"], case["cols"]
        # A few channels carry much larger values than the rest, as a residual stream's do.
        loud = 1 + 30 * (torch.rand((n,), generator=g, device="cuda") < 0.002).float() * torch.rand((n,), generator=g, device="cuda")
        return {"op": "norm", "x": (normal(m, n) * 0.3).to(x), "residual": (normal(m, n) * loud).to(x) if case["residual"] else None,
                "weight": (1 + 0.2 * normal(n)).to(x), "zero": torch.zeros(m, dtype=torch.int8, device="cuda"), "type": x,
                "values": x if x is torch.float16 else torch.float32}    # what dequantize_linear has

    rng = random.Random(seed)
    heads, dim, page, group = case["heads"], case["dim"], case["page"], case.get("group", 4)
    both = _sequences(case)
    rng.shuffle(both)
    lens, new = [s for s, _ in both], [n for _, n in both]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    # The pages of the sequences lie in any order; entries behind a sequence's last page are never looked at.
    wide = max(1, -(-max(lens) // page))
    pages = 1 + sum(-(-s // page) for s in lens)    # the last belongs to nobody
    order = list(range(pages - 1))
    rng.shuffle(order)
    table = []
    for s in lens:
        k = -(-s // page)
        table.append(order[:k] + [-1] * (wide - k))
        order = order[k:]
    s = {"op": case["op"], "type": x, "most": max(new), "rows": cu[-1], "lens": _ints(lens), "table": _ints(table), "page": page,
         "cu": _ints(cu) if min(new) < max(new) else None, "starts": _ints(cu)}
    # Keys have loud channels, and some heads' values are far smaller than others'.
    for name in ("k", "v"):
        loud = 1 + 6 * (torch.rand((heads, 1, dim), generator=g, device="cuda") < 0.03).float() if name == "k" else \
            torch.exp(0.7 * normal(heads, 1, 1))
        spread = torch.exp(0.3 * normal(pages, heads, 1, 1)) * loud
        values = normal(pages, heads, page, dim) * spread
        scale = values.abs().amax(dim=(2, 3)) / 127
        s[name] = torch.round(values / scale[:, :, None, None]).to(torch.int8)
        s[name + "_scale"] = scale
    # Queries, keys and values of the new tokens come out of one product: rows of (group + 2) x heads x dim.
    qkv = normal(cu[-1], (group + 2) * heads, dim)
    qkv[:, : group * heads] *= torch.exp(0.5 * normal(1, group * heads, 1))
    qkv = qkv.to(x)
    s["q"], s["new_k"], s["new_v"] = qkv[:, : group * heads], qkv[:, group * heads: -heads], qkv[:, -heads:]
    s |= {"window": case.get("window", 0), "sinks": case.get("sinks", 0)}
    return s


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


def _own(s):
    from nnops_b200 import ops
    if s["op"] == "norm":
        made = ops.rms_norm_i8(s["x"], s["weight"], residual=s["residual"], eps=_EPS)
        return (ops.dequantize_linear(made[0], made[1], s["zero"], axis=-1, out_dtype=s["values"]), *made[1:])
    cache = s.get("cache")
    if cache is None:
        cache = s["cache"] = ops.CacheI8(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["op"] == "attention":
        return ops.attention_i8_cache(s["q"], cache, s["table"], s["lens"], cu=s["cu"], window=s["window"], sinks=s["sinks"])
    if s["op"] == "write":
        ops.cache_write_i8(cache, s["new_k"], s["new_v"], s["table"], s["lens"], cu=s["cu"])
    values = ops.cache_read_i8(cache, s["table"], s["lens"], rows=s["rows"], cu=s["cu"], out_dtype=s["type"])
    return _written(s, values) if s["op"] == "write" else values


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    t = h * s["weight"].float()
    top = t.abs().amax(dim=1, keepdim=True)
    codes = torch.round(t * (torch.full_like(top, 127.0) / top))
    scale = (top.double() * torch.rsqrt(h.double().square().mean(dim=1, keepdim=True) + _EPS) / 127).float()
    out = ((codes * scale).to(s["values"]), scale[:, 0])
    return out if s["residual"] is None else (*out, h.to(s["type"]))


def _places(s):
    """Of each new row: its sequence, its place among that one's new rows, and its position."""
    row = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"][1:], row, right=True)
    place = row - s["starts"][seq]
    return seq, place, s["lens"][seq] - (s["starts"][seq + 1] - s["starts"][seq]) + place


def _plain_read(s):
    seq, _, pos = _places(s)
    there = (pos >= 0)[:, None, None]
    pos = pos.clamp(min=0)
    page = s["table"][seq, pos // s["page"]].clamp(min=0)
    at = pos % s["page"]
    return tuple(torch.where(there, s[n][page, :, at].float() * s[n + "_scale"][page][:, :, None], 0.0).to(s["type"]) for n in ("k", "v"))


def _plain_write(s):
    seq, place, pos = _places(s)
    there = pos >= 0
    spare, size = s["k"].shape[0] - 1, s["page"]
    pos = pos.clamp(min=0)
    page, at = torch.where(there, s["table"][seq, pos // size].long(), spare), pos % size
    # The pages that get new tokens, as many places for each sequence as the longest run of them can touch.
    new = s["starts"][1:] - s["starts"][:-1]
    first = (s["lens"] - new).clamp(min=0)
    slot = first[:, None] // size + torch.arange((s["most"] + size - 2) // size + 1, device="cuda")
    touched = (slot * size < s["lens"][:, None]) & (new > 0)[:, None]
    ids = torch.where(touched, s["table"].gather(1, slot.clamp(max=s["table"].shape[1] - 1)).long(), spare)
    begins = (slot * size >= first[:, None])[..., None]    # nothing of the page was there before
    for name in ("k", "v"):
        x, codes, scales = s["new_" + name].float(), s[name], s[name + "_scale"]
        top = torch.zeros_like(scales).index_reduce_(0, page, x.abs().amax(dim=2), "amax")[ids]
        need = (top / torch.full_like(top, 127.0)).clamp(min=_LEAST)
        before = scales[ids]
        after = torch.where(touched[..., None], torch.where(begins, need, torch.maximum(before, need)), before)
        held = codes[ids]
        grown = torch.round(held.float() * (before / after)[..., None, None]).to(torch.int8)    # what was there, in the new scale
        codes[ids] = torch.where((touched[..., None] & ~begins)[..., None, None], grown, held)
        scales[ids] = after
        inv = (torch.ones_like(scales) / scales)[page][:, :, None]
        codes[page, :, at] = torch.where(there[:, None, None], torch.round(x * inv).clamp(-127, 127).to(torch.int8), codes[page, :, at])
    return _written(s, _plain_read(s))


def _written(s, values):
    return (*values, s["k_scale"], s["v_scale"], s["k"], s["v"])


def _plain_attention(s):
    seq, place, pos = _places(s)
    heads, dim = s["k"].shape[1], s["k"].shape[3]
    seqs, group = s["table"].shape[0], s["q"].shape[1] // heads
    table = s["table"].clamp(min=0).long()
    k, v = ((s[n][table].float() * s[n + "_scale"][table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(seqs, heads, -1, dim) for n in ("k", "v"))
    q = torch.zeros((seqs, s["most"], heads * group, dim), device="cuda")
    q[seq, place] = s["q"].float()
    at = torch.full((seqs, s["most"]), -1, dtype=torch.int32, device="cuda")
    at[seq, place] = pos
    q = q.view(seqs, s["most"], heads, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, heads, s["most"] * group, dim)
    p = torch.matmul(q, k.transpose(2, 3)).mul_(1 / math.sqrt(dim)).view(seqs, heads, s["most"], group, -1)
    key = torch.arange(k.shape[2], device="cuda", dtype=torch.int32)
    hidden = key > at[..., None]
    if s["window"]:
        hidden |= (key <= at[..., None] - s["window"]) & (key >= s["sinks"])
    hidden = hidden[:, None, :, None]
    p.masked_fill_(hidden, -math.inf)
    p.sub_(p.amax(dim=-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = p.sum(dim=-1)
    o = torch.matmul(p.view(seqs, heads, -1, k.shape[2]), v).view(seqs, heads, s["most"], group, dim)
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
    return o.permute(0, 2, 1, 3, 4).reshape(seqs, s["most"], heads * group, dim)[seq, place].to(s["type"])


_PLAIN = {"norm": _plain_norm, "write": _plain_write, "read": _plain_read, "attention": _plain_attention}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "norm":
        h = s["x"].double() + (s["residual"].double() if s["residual"] is not None else 0)
        y = h / torch.sqrt((h * h).mean(1) + _EPS)[:, None] * s["weight"].double()
        scale = y.abs().amax(1) / 127
        # A code next to a border is either of its neighbours: what it stands for has no exact value.
        return (None, scale) if s["residual"] is None else (None, scale, h)
    if s["op"] == "write":
        return None    # rounded to codes in a fixed order of roundings
    lens, starts, page = s["lens"].tolist(), s["starts"].tolist(), s["page"]
    got = []
    for b, length in enumerate(lens):
        first, last = starts[b], starts[b + 1]
        if last == first:
            continue
        ids = s["table"][b, : -(-length // page)].long()
        kv = []
        for name in ("k", "v"):
            x = s[name][ids].double() * s[name + "_scale"][ids].double()[..., None, None]
            kv.append(x.transpose(1, 2).flatten(0, 1)[:length])    # [tokens, heads, dim]
        if s["op"] == "read":
            lost = last - first - length
            got.append([torch.cat([x.new_zeros(max(0, lost), *x.shape[1:]), x[max(0, -lost):]]) for x in kv])
            continue
        q = s["q"][first:last].double()
        heads = kv[0].shape[1]
        group = q.shape[1] // heads
        o = torch.zeros_like(q)
        step = max(1, int(1.5e8 // max(1, length * group)))
        for i in range(0, q.shape[0], step):
            pos = torch.arange(i, min(i + step, q.shape[0]), device="cuda") + (length - q.shape[0])
            j = torch.arange(length, device="cuda")
            seen = j[None] <= pos[:, None]
            if s["window"]:
                seen &= (j[None] > pos[:, None] - s["window"]) | (j[None] < s["sinks"])
            for h in range(heads):
                if length == 0:
                    continue
                z = torch.einsum("ngd,jd->ngj", q[i:i + step, h * group:(h + 1) * group], kv[0][:, h]) / math.sqrt(q.shape[2])
                z = torch.where(seen[:, None], z, -math.inf)
                w = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
                o[i:i + step, h * group:(h + 1) * group] = torch.einsum("ngj,jd->ngd", w, kv[1][:, h])
        got.append(o)
    if s["op"] == "read":
        return tuple(torch.cat([x[i] for x in got]) for i in range(2))
    return torch.cat(got)
