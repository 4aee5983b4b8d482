"""What the paged key / value cache of ``kch_b200`` is measured on: ``PagedKVCache.append_step`` (rows quantised as they are
written), ``read_step`` (rows read back) and ``forward_step`` (attention of new tokens over the pages).

A batch is ragged: sequence b has ``new_b`` tokens in this call behind ``past_b`` that the cache holds already; its tokens are
consecutive rows of the packed tensors, its pages are scattered over the pool.  A case gives the ends of the ranges of ``new``
and ``past``; the sequences' own lengths are spread over them.  Three kinds of pass:

``write``   new rows into the pages; the 8-bit kinds are read back as the values that they stand for
``read``    rows of a prefix out of the pages, as a session that moves to another process takes them
``attend``  attention of the new tokens' queries over everything the pages hold of their sequences, themselves included

Head counts and widths are those of the stack's two geometries (16 heads of 128, 4 heads of 64), with 1 to 16 key heads.
"""
from __future__ import annotations

import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
QUANT = {"fp8": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}
TINY = 2.0 ** -126


def _case(op, B, new, past, *, dtype="bf16", kind="none", nh=16, n_kv=4, c=128, page=16, window=0, sink=False, name=None):
    case = {"op": op, "B": B, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0], "past_hi": past[1], "dtype": dtype, "kind": kind,
            "nh": nh, "n_kv": n_kv, "c": c, "page": page, "window": window, "sink": sink}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one token each of 64 running sequences goes into an fp8 cache
        _case("write", 64, (1, 1), (100, 8000), kind="fp8", page=16, name="write step fp8"),
        # four prompts of up to 8192 tokens, stored as they are
        _case("write", 4, (6001, 8192), (0, 0), n_kv=8, page=64, name="write prompts bf16"),
        # chunks of seven sequences, fp32 activations, pages that begin and end inside a chunk
        _case("write", 7, (33, 1999), (5, 777), dtype="fp32", kind="int8", nh=4, n_kv=4, c=64, page=32, name="write chunks int8"),
        # a prefix of 32768 tokens leaves an fp8 cache with its session
        _case("read", 1, (32768, 32768), (0, 0), kind="fp8", n_kv=8, page=64, name="read prefix fp8"),
        # the last rows of 24 sequences, at odd offsets
        _case("read", 24, (1, 257), (3, 3001), dtype="fp32", kind="int8", n_kv=2, c=64, page=16, name="read tails int8"),
        # one token of one short conversation: launches and latency
        _case("attend", 1, (1, 1), (200, 200), page=16, name="step of one sequence"),
        # a decode step of 64 sequences of 500 to 16000 tokens
        _case("attend", 64, (1, 1), (500, 16000), n_kv=4, page=16, name="step of 64 sequences"),
        # the same from an fp8 cache, a single key head, a sink in the denominator
        _case("attend", 64, (1, 1), (500, 16000), kind="fp8", n_kv=1, page=64, sink=True, name="step of 64 fp8 mqa"),
        # one long sequence: the split of the key axis carries it
        _case("attend", 1, (4, 4), (131001, 131001), kind="int8", n_kv=2, page=32, name="four tokens over 131005 int8"),
        # running sequences and chunks of prompts in one call, a window of 1000 tokens, groups of three heads
        _case("attend", 24, (1, 511), (7, 3500), kind="fp8", nh=12, n_kv=4, page=16, window=1000, sink=True, name="mixed batch fp8 window"),
        # fp32, the small geometry
        _case("attend", 3, (200, 700), (0, 1500), dtype="fp32", nh=4, n_kv=2, c=64, page=32, name="chunks fp32"),
        # a chunk of 4096 tokens of a long prompt behind the 28672 before it
        _case("attend", 1, (4096, 4096), (28672, 28672), n_kv=4, page=128, name="chunk of 4096 at 28672"),
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def _range(rng, lo, hi):
    a, b = sorted((_between(rng, lo, hi), _between(rng, lo, hi)))
    return a, b


def draw(rng):
    top = {}
    for case in listed():
        w = work(case)
        op = case["op"]
        top[op] = (max(top.get(op, (0, 0))[0], w["bytes"]), max(top.get(op, (0, 0))[1], w["flops"]))
    while True:
        op = rng.choice(("write", "read", "attend", "attend", "attend"))
        c = rng.choice((64, 128, 128))
        nh = 4 if c == 64 else rng.choice((12, 16, 16))
        n_kv = rng.choice([n for n in (1, 2, 4, 8, 16) if nh % n == 0])
        dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
        kind = rng.choice(("none", "none", "fp8", "int8"))
        B = _between(rng, 1, 64)
        new = _range(rng, 1, 8192 if op != "attend" else rng.choice((1, 8, 600, 4096)))
        past = _range(rng, 1, 2000 if op != "attend" else 131072 if dtype == "bf16" else 4000)
        window = rng.choice((0, 0, 0, 128, 1000)) if op == "attend" else 0
        case = _case(op, B, new, past, dtype=dtype, kind=kind, nh=nh, n_kv=n_kv, c=c, page=rng.choice((16, 16, 32, 64, 128)), window=window,
                     sink=op == "attend" and rng.random() < 0.3)
        w = work(case)
        # (the plain form pads the batch: its scores have to fit as well)
        scores = B * nh * new[1] * (new[1] + past[1]) if op == "attend" else 0
        rows = B * n_kv * c * (new[1] + past[1])
        flops = w["flops"] * (16 if dtype == "fp32" else 1)
        if w["bytes"] <= top[op][0] and flops <= top[op][1] and scores <= 2 ** 31 and rows <= 2 ** 30:
            return case


def _spread(lo, hi, n, step):
    """n lengths over lo .. hi: the longest first, the others at multiples of `step` of the range, taken round."""
    return [round(hi - (hi - lo) * ((i * step) % 1.0)) for i in range(n)]


def _lengths(case):
    return (_spread(case["new_lo"], case["new_hi"], case["B"], 0.6180339887498949),
            _spread(case["past_lo"], case["past_hi"], case["B"], 0.7548776662466927))


def _sees(case, new, past):
    """How many keys the queries of a sequence see together, and how many different ones."""
    w = case["window"]
    if not w:
        return new * past + new * (new + 1) // 2, past + new
    full = max(0, min(new, past + new - w + 1) if past < w else new)      # queries that see a whole window
    ramp = new - full
    return full * w + ramp * past + ramp * (ramp + 1) // 2, min(past + new, new + w - 1)


def work(case):
    new, past = _lengths(case)
    c, n_kv, nh = case["c"], case["n_kv"], case["nh"]
    es = 2 if case["dtype"] == "bf16" else 4
    row = 2 * n_kv * (c * es if case["kind"] == "none" else c + 4)       # a token in the pages
    act = 2 * n_kv * c * es                                             # a token's k and v as activations
    if case["op"] == "write":      # read the rows, write the pages (the 8-bit kinds: and the values that they stand for)
        return {"bytes": sum(new) * (act + row + (0 if case["kind"] == "none" else act)), "flops": 0}
    if case["op"] == "read":
        return {"bytes": sum(new) * (act + row), "flops": 0}
    seen = [_sees(case, n, p) for n, p in zip(new, past)]
    return {"bytes": sum(s[1] for s in seen) * row + 2 * sum(new) * nh * c * es, "flops": 4 * c * nh * sum(s[0] for s in seen)}


def _handle(s):
    """The cache object over the pool of this state."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kda-csa-hca-fusion_b200"))
    import kch_b200
    case = s["case"]
    return kch_b200.PagedKVCache(s["k_pages"].shape[0], case["page"], case["n_kv"], case["c"], DEV, DTYPES[case["dtype"]],
                                 kv_quant=None if case["kind"] == "none" else case["kind"],
                                 storage=(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    new, past = _lengths(case)
    B, page, n_kv, c, dtype = case["B"], case["page"], case["n_kv"], case["c"], DTYPES[case["dtype"]]
    held = [-(-(n + p) // page) for n, p in zip(new, past)]              # pages of a sequence
    pool = sum(held) + 3
    ids = torch.randperm(pool, generator=g, device=DEV)[:sum(held)].to(torch.int32)
    table = torch.full((B, max(held)), -1, dtype=torch.int32, device=DEV)
    table[torch.arange(max(held), device=DEV) < torch.tensor(held, device=DEV)[:, None]] = ids
    rows = (pool, n_kv, page, c)
    s = {"case": case, "new": new, "past": past, "table": table,
         "t0": torch.tensor(past, dtype=torch.int32, device=DEV),
         "cu": torch.tensor([sum(new[:i]) for i in range(B + 1)], dtype=torch.int32, device=DEV)}
    for x in ("k", "v"):                                                # what earlier calls have left in the pages
        if case["kind"] == "none":
            s[x + "_pages"], s[x + "_scales"] = torch.randn(rows, generator=g, device=DEV, dtype=dtype), None
        else:
            s[x + "_pages"], s[x + "_scales"] = _quantise(torch.randn(rows, generator=g, device=DEV, dtype=dtype), case["kind"])
    if case["op"] == "write":
        for x in ("k", "v"):
            s[x] = torch.randn(sum(new), n_kv, c, generator=g, device=DEV, dtype=dtype)
    if case["op"] == "attend":
        s["q"] = torch.randn(sum(new), case["nh"], c, generator=g, device=DEV, dtype=dtype)
        s["sink"] = torch.randn(case["nh"], generator=g, device=DEV) if case["sink"] else None
    if own:
        s["cache"] = _handle(s)
    return s


def _quantise(x, kind):
    """A scale per row: its largest value over the largest that the type holds, kept in 32 bits; the row over its scale, rounded
    (in 64 bits: a quotient next to the middle between two values of the type would fall on it in 32)."""
    store, most = QUANT[kind]
    amax = x.double().abs().amax(-1)
    scale = torch.where(amax > 0, (amax / most).clamp_min(TINY), 1.0).float()
    x = x.double() / scale.double()[..., None]
    if kind == "fp8":      # e4m3: 4 bits from the leading one on, steps of 2^-9 at least
        step = torch.ldexp(torch.ones_like(x), (torch.frexp(x)[1] - 4).clamp_min(-9))
        return (torch.round(x / step) * step).clamp(-most, most).to(store), scale
    return torch.round(x).to(store), scale


def _sites(s):
    """Of every packed row: its sequence, and its page and row there."""
    cu, page = s["cu"].long(), s["case"]["page"]
    n = sum(s["new"])
    seq = torch.searchsorted(cu[1:], torch.arange(n, device=DEV), right=True)
    pos = s["t0"].long()[seq] + torch.arange(n, device=DEV) - cu[seq]
    return s["table"].long()[seq, pos // page], pos % page


def _values(pages, scales, at):
    """Rows of the pages as fp32 values: [..., n_kv, c]."""
    x = pages[at[0], :, at[1]].float()
    return x if scales is None else x * scales[at[0], :, at[1]][..., None]


def _write(s):
    at = _sites(s)
    for x in ("k", "v"):
        if s["case"]["kind"] == "none":
            s[x + "_pages"][at[0], :, at[1]] = s[x]
        else:
            payload, scale = _quantise(s[x], s["case"]["kind"])
            s[x + "_pages"].view(torch.uint8)[at[0], :, at[1]] = payload.view(torch.uint8)
            s[x + "_scales"][at[0], :, at[1]] = scale


def _read(s):
    at, dtype = _sites(s), DTYPES[s["case"]["dtype"]]
    return [_values(s[x + "_pages"], s[x + "_scales"], at).to(dtype) for x in ("k", "v")]


def _attend(s):
    case = s["case"]
    page, nh, n_kv, c = case["page"], case["nh"], case["n_kv"], case["c"]
    new, total = max(s["new"]), max(n + p for n, p in zip(s["new"], s["past"]))
    cu, t0 = s["cu"].long(), s["t0"].long()
    # queries padded to [B, n_kv, new, G, c], keys and values to [B, n_kv, total, c]
    tok = torch.arange(new, device=DEV)
    here = tok < (cu[1:] - cu[:-1])[:, None]
    q = s["q"].float()[torch.where(here, cu[:-1, None] + tok, 0)].view(-1, new, n_kv, nh // n_kv, c).transpose(1, 2)
    pos = torch.arange(total, device=DEV)
    at = s["table"].long().clamp_min(0)[:, pos // page], (pos % page).expand(case["B"], total)
    k, v = (_values(s[x + "_pages"], s[x + "_scales"], at).transpose(1, 2) for x in ("k", "v"))
    logits = (q.flatten(2, 3) * c ** -0.5) @ k.transpose(2, 3)           # [B, n_kv, new * G, total]
    p = (t0[:, None] + tok)[:, :, None]
    seen = (pos <= p) & (pos > p - case["window"] if case["window"] else pos <= p)
    logits = logits.view(-1, n_kv, new, nh // n_kv, total).masked_fill_(~seen[:, None, :, None], float("-inf"))
    top = logits.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(n_kv, 1, nh // n_kv, 1)
        top = torch.maximum(top, sink)
    e = logits.sub_(top).exp_()
    below = e.sum(-1, keepdim=True)
    if s["sink"] is not None:
        below = below + (sink - top).exp()
    out = (e.flatten(2, 3) @ v).view(-1, n_kv, new, nh // n_kv, c) / below
    return out.transpose(1, 2).reshape(-1, new, nh, c)[here].to(s["q"].dtype)


def run(state):
    s = state
    op, kind = s["case"]["op"], s["case"]["kind"]
    if own:
        cache, batch = s["cache"], (s["table"], s["t0"], s["cu"])
        if op == "attend":
            return cache.forward_step(s["q"], *batch, sink_logits=s["sink"], sliding_window=s["case"]["window"])
        if op == "write":
            cache.append_step(s["k"], s["v"], *batch)
            return [s["k_pages"], s["v_pages"]] if kind == "none" else list(cache.read_step(*batch, n_rows=s["k"].shape[0]))
        return list(cache.read_step(*batch, n_rows=sum(s["new"])))
    if op == "attend":
        return _attend(s)
    if op == "write":
        _write(s)
        return [s["k_pages"], s["v_pages"]] if kind == "none" else _read(s)
    return _read(s)


def _nearest(x, kind):
    """The nearest of the values that the type holds, and the one with the even code in the middle between two."""
    store, most = QUANT[kind]
    codes = torch.arange(int(most) + 1 if kind == "int8" else 127, device=DEV)
    held = codes.to(torch.uint8).view(store).double()                    # 0 and the positive ones, in order
    size = x.abs()
    above = torch.searchsorted(held, size).clamp_(1, len(held) - 1)
    low, high = size - held[above - 1], held[above] - size
    up = (high < low) | ((high == low) & (above % 2 == 0))
    return torch.where(up, held[above], held[above - 1]).copysign(x)


def exact(case, seed):
    s = prepare(case, seed)
    page, B, kind = case["page"], case["B"], case["kind"]
    ends = [sum(s["new"][:b + 1]) for b in range(B)]
    if case["op"] == "write" and kind == "none":       # a copy: every value as it was
        _write(s)
        return [s["k_pages"].double(), s["v_pages"].double()]
    outs = []
    if case["op"] == "write":
        for x in (s["k"].double(), s["v"].double()):
            amax = x.abs().amax(-1, keepdim=True)
            most = QUANT[kind][1]
            scale = torch.where(amax > 0, (amax / most).float().double(), 1.0)     # kept in 32 bits
            outs.append(_nearest(x / scale, kind) * scale)
        return outs

    def rows(x, b, first, last):
        """Rows first .. last of sequence b, [n_kv, last - first, c]."""
        got = s[x + "_pages"][s["table"][b, :-(-last // page)].long()].double()
        if kind != "none":
            got = got * s[x + "_scales"][s["table"][b, :-(-last // page)].long()].double()[..., None]
        return got.transpose(0, 1).flatten(1, 2)[:, first:last]

    if case["op"] == "read":
        return [torch.cat([rows(x, b, s["past"][b], s["past"][b] + s["new"][b]).transpose(0, 1) for b in range(B)]) for x in ("k", "v")]
    group = case["nh"] // case["n_kv"]
    for b in range(B):
        n, p = s["new"][b], s["past"][b]
        k, v = (rows(x, b, 0, p + n) for x in ("k", "v"))
        q = s["q"][ends[b] - n:ends[b]].double()
        far = torch.arange(p, p + n, device=DEV)[:, None] - torch.arange(p + n, device=DEV)      # how far back a key lies
        hidden = (far < 0) | (far >= case["window"]) if case["window"] else far < 0
        heads = []
        for h in range(case["nh"]):
            l = (q[:, h] @ k[h // group].T / case["c"] ** 0.5).masked_fill_(hidden, float("-inf"))
            z = torch.logsumexp(l, 1, keepdim=True)
            if s["sink"] is not None:
                z = torch.logaddexp(z, s["sink"][h].double().expand_as(z))
            heads.append(l.sub_(z).exp_() @ v[h // group])
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)
