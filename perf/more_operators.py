"""What a prompt needs beside the paged cache of ``kch_b200``, measured: its queries and keys turned by their positions
(``RotaryPositions.rotate``), attended as a whole (``prompt_attention``), kept in 4 bits and attended there
(``PagedKVCache(kv_quant="int4")``: ``append_step``, ``read_step``, ``forward_step``).

A batch is ragged and packed: the tokens of a sequence are consecutive rows.  A case gives the ends of the ranges of new and earlier
tokens; the sequences' own lengths are spread over them.  Five kinds of pass:

``rotate``  queries and keys, column slices of a fused projection, turned by positions on one to three axes
``prompt``  causal attention of packed prompts, queries, keys and values column slices of a fused projection
``write``   new rows into the pages in 4 bits, read back as the values that they stand for
``read``    rows of the pages, as a session that moves to another process takes them
``attend``  attention of new tokens' queries over everything the pages hold of their sequences, themselves included

Head counts and widths are those of the stack's two geometries (16 heads of 128, 4 heads of 64), with 1 to 16 key heads.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
GROUP = 32                  # channels that share a scale in 4 bits


def _case(op, B, new, past=(0, 0), *, dtype="bf16", nh=16, n_kv=4, c=128, page=16, window=0, sink=False, axes=1, turned=0, neighbours=False,
          back=False, name=None):
    case = {"op": op, "B": B, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0], "past_hi": past[1], "dtype": dtype, "nh": nh, "n_kv": n_kv,
            "c": c, "page": page, "window": window, "sink": sink, "axes": axes, "turned": turned or c, "neighbours": neighbours, "back": back}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # a decode step of 64 sequences: latency
        _case("rotate", 64, (1, 1), (100, 30000), name="rotate step"),
        # prompts of text and pictures, positions on three axes
        _case("rotate", 6, (2000, 6100), (0, 0), n_kv=8, axes=3, name="rotate prompts three axes"),
        # fp32, neighbouring channels, half of a head turned, turned back (the gradient of it)
        _case("rotate", 9, (33, 999), (5, 70000), dtype="fp32", nh=4, n_kv=4, c=64, axes=2, turned=32, neighbours=True, back=True,
              name="rotate back fp32 half"),
        # one short question: launches and latency
        _case("prompt", 1, (100, 100), name="prompt of 100"),
        # a batch of prompts of all lengths, groups of three heads, a window, a sink
        _case("prompt", 40, (1, 1500), nh=12, n_kv=4, window=700, sink=True, name="prompts ragged window"),
        # two long documents
        _case("prompt", 2, (8300, 14001), n_kv=2, name="prompts long"),
        # fp32, the small geometry
        _case("prompt", 5, (50, 900), dtype="fp32", nh=4, n_kv=2, c=64, name="prompts fp32"),
        # four prompts stored
        _case("write", 4, (4001, 8192), n_kv=8, page=64, name="write prompts"),
        # the last rows of 24 sequences, at odd offsets, as fp32
        _case("read", 24, (1, 257), (3, 3001), dtype="fp32", n_kv=2, c=64, name="read tails"),
        # a decode step of 64 sequences of 500 to 16000 tokens
        _case("attend", 64, (1, 1), (500, 16000), page=32, name="step of 64"),
        # four tokens of one long sequence, one key head, a sink: the split of the key axis carries it
        _case("attend", 1, (4, 4), (131001, 131001), n_kv=1, page=64, sink=True, name="four tokens over 131005"),
        # running sequences and chunks of prompts in one call
        _case("attend", 12, (1, 2048), (5, 12000), n_kv=4, page=16, name="chunks and steps"),
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
    top["read"] = (top["write"][0] // 2, 0)
    while True:
        op = rng.choice(("rotate", "rotate", "prompt", "prompt", "prompt", "write", "read", "attend", "attend", "attend"))
        c = rng.choice((64, 128, 128))
        nh = 4 if c == 64 else rng.choice((12, 16, 16))
        n_kv = rng.choice([n for n in (1, 2, 4, 8, 16) if nh % n == 0])
        dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
        B = _between(rng, 1, 64)
        new = _range(rng, 1, {"rotate": 30000, "prompt": 14000, "attend": rng.choice((1, 8, 600, 4096))}.get(op, 8192))
        past = (0, 0) if op == "prompt" else _range(rng, 1, {"rotate": 1000000, "attend": 131072 if dtype == "bf16" else 4000}.get(op, 3000))
        attends = op in ("prompt", "attend")
        window = rng.choice((0, 0, 0, 128, 1000)) if attends else 0
        axes = rng.choice((1, 1, 2, 3)) if op == "rotate" else 1
        turned = rng.choice((c, c, c // 2)) if op == "rotate" else c
        case = _case(op, B, new, past, dtype=dtype, nh=nh, n_kv=n_kv, c=c, page=rng.choice((16, 16, 32, 64, 128)), window=window,
                     sink=attends and rng.random() < 0.3, axes=axes, turned=turned, neighbours=op == "rotate" and rng.random() < 0.3,
                     back=op == "rotate" and rng.random() < 0.3)
        w = work(case)
        # (the plain form pads the batch: its scores have to fit as well)
        total = new[1] + past[1]
        scores = B * nh * new[1] * total if attends else 0
        rows = B * n_kv * c * total if attends else 0
        flops = w["flops"] * (16 if dtype == "fp32" else 1)
        if w["bytes"] <= top[op][0] and (flops <= top[op][1] or not attends) and scores <= 2 ** 33 and rows <= 2 ** 30:
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
    row = 2 * n_kv * (c // 2 + 2 * (c // GROUP))                          # a token in the pages
    act = 2 * n_kv * c * es                                             # a token's k and v as activations
    if case["op"] == "rotate":     # read, turn and write (a sine and a cosine are 1 each)
        return {"bytes": sum(new) * (2 * (nh + n_kv) * c * es + 4 * case["axes"]), "flops": sum(new) * (3 * (nh + n_kv) + 2) * case["turned"]}
    if case["op"] == "write":      # read the rows, write the pages and the values that they stand for
        return {"bytes": sum(new) * (act + row + act), "flops": 0}
    if case["op"] == "read":
        return {"bytes": sum(new) * (act + row), "flops": 0}
    seen = [_sees(case, n, p) for n, p in zip(new, past)]
    flops = 4 * c * nh * sum(s[0] for s in seen)
    if case["op"] == "prompt":
        return {"bytes": sum(new) * (act + 2 * nh * c * es), "flops": flops}
    return {"bytes": sum(s[1] for s in seen) * row + 2 * sum(new) * nh * c * es, "flops": flops}


def _sections(case):
    """Pairs of channels on each axis: a quarter of them time's, the others' the rest."""
    pairs, axes = case["turned"] // 2, case["axes"]
    first = pairs if axes == 1 else pairs // 4
    rest = [(pairs - first) // (axes - 1)] * (axes - 1) if axes > 1 else []
    return (pairs - sum(rest), *rest)


def _handle(s):
    """The framework's object that a program keeps over calls."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kda-csa-hca-fusion_b200"))
    import kch_b200
    case = s["case"]
    if case["op"] == "rotate":
        return kch_b200.RotaryPositions(case["c"], DEV, rotary_dim=case["turned"], sections=_sections(case), neighbours=case["neighbours"])
    if case["op"] == "prompt":
        return kch_b200.prompt_attention
    return kch_b200.PagedKVCache(s["k_pages"].shape[0], case["page"], case["n_kv"], case["c"], DEV, DTYPES[case["dtype"]], kv_quant="int4",
                                 storage=(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    new, past = _lengths(case)
    B, page, n_kv, nh, c, dtype = case["B"], case["page"], case["n_kv"], case["nh"], case["c"], DTYPES[case["dtype"]]
    s = {"case": case, "new": new, "past": past,
         "t0": torch.tensor(past, dtype=torch.int32, device=DEV),
         "cu": torch.tensor([sum(new[:i]) for i in range(B + 1)], dtype=torch.int32, device=DEV)}
    n = sum(new)
    if case["op"] in ("rotate", "prompt"):
        both = torch.randn(n, (nh + 2 * n_kv) * c, generator=g, device=DEV, dtype=dtype)
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, c)) for x in both.split((nh * c, n_kv * c, n_kv * c), 1))
    if case["op"] == "rotate":
        seq = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(new, device=DEV))
        at = torch.arange(n, device=DEV) - s["cu"].long()[seq]
        # text and pictures in turns of 256 tokens: a picture's stand still in time, 16 x 16 of them in height and width
        text, place = (at // 256) % 2 == 0, at % 256
        time = torch.where(text, at, at - place) + s["t0"].long()[seq]
        axes = [time, torch.where(text, time, place // 16 + time), torch.where(text, time, place % 16 + time)]
        s["positions"] = torch.stack(axes[:case["axes"]], 1).to(torch.int32)
    if case["op"] in ("write", "read", "attend"):
        held = [-(-(x + p) // page) for x, p in zip(new, past)]          # pages of a sequence
        pool = sum(held) + 3
        ids = torch.randperm(pool, generator=g, device=DEV)[:sum(held)].to(torch.int32)
        s["table"] = torch.full((B, max(held)), -1, dtype=torch.int32, device=DEV)
        s["table"][torch.arange(max(held), device=DEV) < torch.tensor(held, device=DEV)[:, None]] = ids
        for x in ("k", "v"):                                            # what earlier calls have left in the pages
            s[x + "_pages"], s[x + "_scales"] = _quantise(torch.randn(pool, n_kv, page, c, generator=g, device=DEV, dtype=dtype))
    if case["op"] == "write":
        for x in ("k", "v"):
            s[x] = torch.randn(n, n_kv, c, generator=g, device=DEV, dtype=dtype)
    if case["op"] == "attend":
        s["q"] = torch.randn(n, nh, c, generator=g, device=DEV, dtype=dtype)
    s["sink"] = torch.randn(nh, generator=g, device=DEV) if case["sink"] else None
    if own:
        s["handle"] = _handle(s)
    return s


def _quantise(x):
    """Bytes of two codes (of the even channel in the low half, 8 more than the code) and a scale for 32 channels: the smallest number
    of 5 bits, of which 7 times is no less than the largest value; the values over it, rounded.  (In 64 bits: a quotient next to the
    middle between two codes would fall on it in 32.)"""
    x = x.double().unflatten(-1, (-1, GROUP))
    amax = x.abs().amax(-1)
    bits, power = torch.frexp(amax / 7)
    scale = torch.where(amax > 0, torch.ldexp(torch.ceil(bits * 32) / 32, power).clamp_min(2.0 ** -126), 1.0)
    codes = (torch.round(x / scale[..., None]) + 8).flatten(-2).to(torch.uint8).unflatten(-1, (-1, 2))
    return codes[..., 0] | codes[..., 1] << 4, scale.to(torch.bfloat16)


def _values(pages, scales):
    """What bytes and scales stand for, [..., c] in 32 bits."""
    codes = torch.stack((pages & 15, pages >> 4), -1).flatten(-2).float() - 8
    return codes * scales.float().repeat_interleave(GROUP, -1)


def _sites(s):
    """Of every packed row: its page and its row there."""
    cu, page = s["cu"].long(), s["case"]["page"]
    n = sum(s["new"])
    seq = torch.searchsorted(cu[1:], torch.arange(n, device=DEV), right=True)
    pos = s["t0"].long()[seq] + torch.arange(n, device=DEV) - cu[seq]
    return s["table"].long()[seq, pos // page], pos % page


def _write(s):
    at = _sites(s)
    for x in ("k", "v"):
        s[x + "_pages"][at[0], :, at[1]], s[x + "_scales"][at[0], :, at[1]] = _quantise(s[x])


def _read(s):
    at, dtype = _sites(s), DTYPES[s["case"]["dtype"]]
    return [_values(s[x + "_pages"][at[0], :, at[1]], s[x + "_scales"][at[0], :, at[1]]).to(dtype) for x in ("k", "v")]


def _rotate(s):
    case = s["case"]
    r, pairs = case["turned"], case["turned"] // 2
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=DEV), torch.tensor(_sections(case), device=DEV))
    freq = 10000.0 ** (torch.arange(pairs, device=DEV, dtype=torch.float64) * (-2.0 / r))
    angle = s["positions"].double()[:, axis] * freq                      # [N, pairs]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if case["back"]:
        sin = -sin
    out = []
    for x in (s["q"], s["k"]):
        y = x.float()
        if case["neighbours"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = y[..., :pairs], y[..., pairs:r]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        out.append(torch.cat((turned, y[..., r:]), -1).to(x.dtype))
    return out


def _attend(s):
    case = s["case"]
    page, nh, n_kv, c, paged = case["page"], case["nh"], case["n_kv"], case["c"], case["op"] == "attend"
    new, total = max(s["new"]), max(n + p for n, p in zip(s["new"], s["past"]))
    cu, t0 = s["cu"].long(), s["t0"].long()
    # queries padded to [B, n_kv, new, G, c], keys and values to [B, n_kv, total, c]
    tok = torch.arange(new, device=DEV)
    here = tok < (cu[1:] - cu[:-1])[:, None]
    rows = torch.where(here, cu[:-1, None] + tok, 0)
    q = s["q"].float()[rows].view(-1, new, n_kv, nh // n_kv, c).transpose(1, 2)
    pos = torch.arange(total, device=DEV)
    if paged:
        at = s["table"].long().clamp_min(0)[:, pos // page], (pos % page).expand(case["B"], total)
        k, v = (_values(s[x + "_pages"][at[0], :, at[1]], s[x + "_scales"][at[0], :, at[1]]).transpose(1, 2) for x in ("k", "v"))
    else:
        k, v = (s[x].float()[rows].transpose(1, 2) for x in ("k", "v"))
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
    op, case = s["case"]["op"], s["case"]
    if own:
        h = s["handle"]
        if op == "rotate":
            return list(h.rotate(s["q"], s["k"], s["positions"], inverse=case["back"]))
        if op == "prompt":
            return h(s["q"], s["k"], s["v"], s["cu"], sink_logits=s["sink"], sliding_window=case["window"])
        batch = (s["table"], s["t0"], s["cu"])
        if op == "attend":
            return h.forward_step(s["q"], *batch, sink_logits=s["sink"], sliding_window=case["window"])
        if op == "write":
            h.append_step(s["k"], s["v"], *batch)
        return list(h.read_step(*batch, n_rows=sum(s["new"])))
    if op == "rotate":
        return _rotate(s)
    if op in ("prompt", "attend"):
        return _attend(s)
    if op == "write":
        _write(s)
    return _read(s)


def exact(case, seed):
    s = prepare(case, seed)
    page, B, nh, n_kv, c = case["page"], case["B"], case["nh"], case["n_kv"], case["c"]
    ends = [sum(s["new"][:b + 1]) for b in range(B)]
    if case["op"] == "rotate":       # as a product of complex numbers, a pair each
        r, base = case["turned"], math.log(10000.0)
        freq = torch.tensor([math.exp(-base * 2 * i / r) for i in range(r // 2)], dtype=torch.float64, device=DEV)
        place = torch.cat([s["positions"][:, a:a + 1].double().expand(-1, n) for a, n in enumerate(_sections(case))], 1)
        turn = torch.polar(torch.ones_like(place), place * freq * (-1 if case["back"] else 1))[:, None]
        first, second = (slice(0, r, 2), slice(1, r, 2)) if case["neighbours"] else (slice(0, r // 2), slice(r // 2, r))
        outs = []
        for x in (s["q"], s["k"]):
            y = x.double().clone()
            z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
            y[..., first], y[..., second] = z.real, z.imag
            outs.append(y)
        return outs
    if case["op"] == "write":
        outs = []
        held = torch.arange(-7, 8, device=DEV, dtype=torch.float64)
        for x in (s["k"].double(), s["v"].double()):
            y = x.view(*x.shape[:2], c // GROUP, GROUP)
            most = y.abs().amax(-1, keepdim=True)
            # candidates: 16 .. 31 times powers of two around a seventh of the largest value; the smallest that reaches it
            power = torch.floor(torch.log2(most / 7)) - 4
            sizes = torch.ldexp(torch.arange(15, 34, device=DEV, dtype=torch.float64), power.expand(*most.shape[:-1], 19))
            scale = torch.where(sizes * 7 >= most, sizes, torch.inf).amin(-1, keepdim=True)
            scale = torch.where(most > 0, scale, 1.0)
            low = torch.searchsorted(held, (y / scale).clamp(-7, 7), right=True).clamp(1, 14) - 1
            under, over = y / scale - held[low], held[low + 1] - y / scale
            up = (over < under) | ((over == under) & (held[low + 1] % 2 == 0))
            outs.append((torch.where(up, held[low + 1], held[low]) * scale).view(x.shape))
        return outs

    def rows(x, b, first, last):
        """Rows first .. last of sequence b, [n_kv, last - first, c]."""
        if case["op"] == "prompt":
            return s[x][ends[b] - s["new"][b]:ends[b]].double().transpose(0, 1)[:, first:last]
        ids = s["table"][b, :-(-last // page)].long()
        got = s[x + "_pages"][ids].transpose(0, 1).flatten(1, 2)[:, first:last].int()
        by = s[x + "_scales"][ids].transpose(0, 1).flatten(1, 2)[:, first:last].double()
        y = torch.empty(*got.shape[:2], c, dtype=torch.float64, device=DEV)
        y[..., 0::2], y[..., 1::2] = got % 16 - 8, got // 16 - 8
        return (y.view(*got.shape[:2], -1, GROUP) * by[..., None]).flatten(2)

    if case["op"] == "read":
        return [torch.cat([rows(x, b, s["past"][b], s["past"][b] + s["new"][b]).transpose(0, 1) for b in range(B)]) for x in ("k", "v")]
    if sum(n * (n + p) for n, p in zip(s["new"], s["past"])) * nh * c > 2 ** 42:
        return None
    group, outs = nh // n_kv, []
    for b in range(B):
        n, p = s["new"][b], s["past"][b]
        k, v = (rows(x, b, 0, p + n) for x in ("k", "v"))
        q = s["q"][ends[b] - n:ends[b]].double()
        far = torch.arange(p, p + n, device=DEV)[:, None] - torch.arange(p + n, device=DEV)      # how far back a key lies
        hidden = (far < 0) | (far >= case["window"]) if case["window"] else far < 0
        heads = []
        for h in range(nh):
            l = (q[:, h] @ k[h // group].T / c ** 0.5).masked_fill_(hidden, float("-inf"))
            z = torch.logsumexp(l, 1, keepdim=True)
            if s["sink"] is not None:
                z = torch.logaddexp(z, s["sink"][h].double().expand_as(z))
            heads.append(l.sub_(z).exp_() @ v[h // group])
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)
