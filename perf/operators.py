"""What a serving step of many ragged sequences does around a model's products, as its speed is measured: keys and values appended to a paged cache
with the norms and the rotation on the way, attention over that cache, and the draw of the next tokens.

``run`` takes the framework's operators where ``own`` is true and plain torch in 32 or 64 bits where it is false; ``exact`` states them once more in
64 bits.  Head layouts, page sizes and vocabularies come from the repository's model presets (20 query heads over 4 of 128 channels, 24 over 4 of 256 with
64 rotated channels, 48 over 8 of 128; 50304 to 262144 tokens); batches and lengths are generic.

A cache: pages ``[pages, kv heads, page, head size]`` for keys and for values, in 16 bits or as e4m3 numbers in units of a power of two for each page and
head; ``table[b, j]`` is the page of positions ``j * page`` and on of sequence ``b``, ``lengths[b]`` its tokens with the new ones, whose rows are
``starts[b] .. starts[b + 1] - 1`` of the operands (without ``starts``: one row each).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
LARGEST, LEAST = 448.0, -100           # of e4m3; the smallest exponent of a page's scale


def listed():
    return [
        # the cache write of one user's next token: nothing but latency
        {"name": "append_one", "kind": "append", "batch": 1, "context": 501, "fresh": 1, "heads": 20, "kv": 4, "dim": 128, "rot": 128, "page": 16, "norm": True,
         "cache": "e4m3", "dtype": "bf16"},
        # a decoding step of a full batch
        {"name": "append_batch", "kind": "append", "batch": 64, "context": 2000, "fresh": 1, "heads": 48, "kv": 8, "dim": 128, "rot": 128, "page": 64, "norm": True,
         "cache": "e4m3", "dtype": "bf16"},
        # pieces of prompts of ragged length between decoding steps, heads of 256 of which a quarter turns, 16-bit pages
        {"name": "append_chunk", "kind": "append", "batch": 9, "context": 3001, "fresh": 333, "heads": 24, "kv": 4, "dim": 256, "rot": 64, "page": 32, "norm": True,
         "cache": "fp16", "dtype": "fp16"},
        # whole prompts
        {"name": "append_prompt", "kind": "append", "batch": 8, "context": 4096, "fresh": 4096, "heads": 48, "kv": 8, "dim": 128, "rot": 128, "page": 64, "norm": False,
         "cache": "e4m3", "dtype": "bf16"},
        # one user's next token in a short chat
        {"name": "attend_one", "kind": "attend", "batch": 1, "context": 501, "fresh": 1, "heads": 20, "kv": 4, "dim": 128, "page": 16, "window": 0,
         "cache": "e4m3", "dtype": "bf16"},
        # a decoding step of a batch of chats, heads of 256
        {"name": "attend_batch", "kind": "attend", "batch": 32, "context": 2000, "fresh": 1, "heads": 24, "kv": 4, "dim": 256, "page": 32, "window": 0,
         "cache": "e4m3", "dtype": "bf16"},
        # a decoding step over long documents
        {"name": "attend_long", "kind": "attend", "batch": 32, "context": 16384, "fresh": 1, "heads": 48, "kv": 8, "dim": 128, "page": 64, "window": 0,
         "cache": "e4m3", "dtype": "bf16"},
        # pieces of prompts of ragged length against what their sequences hold, 16-bit pages
        {"name": "attend_chunk", "kind": "attend", "batch": 6, "context": 3001, "fresh": 250, "heads": 20, "kv": 4, "dim": 128, "page": 16, "window": 0,
         "cache": "bf16", "dtype": "bf16"},
        # one user's next token, with the usual settings
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 151936, "dtype": "fp32", "filter": "k50p"},
        # a batch of requests that each bring their own settings
        {"name": "sample_mixed", "kind": "sample", "rows": 33, "vocab": 248320, "dtype": "bf16", "filter": "mixed"},
        # completions sampled for training: no filter
        {"name": "sample_plain", "kind": "sample", "rows": 256, "vocab": 50304, "dtype": "fp32", "filter": "none"},
        # a large batch over the largest vocabulary, cut by mass alone
        {"name": "sample_large", "kind": "sample", "rows": 128, "vocab": 262144, "dtype": "fp32", "filter": "p"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "sample"))
    if kind == "sample":
        vocab = _log(rng, 500, 262144)
        return {"kind": kind, "rows": _log(rng, 1, min(512, 2 ** 25 // vocab)), "vocab": vocab, "dtype": rng.choice(("fp32", "bf16", "fp16")),
                "filter": rng.choice(("none", "p", "k50p", "min", "mixed"))}
    heads, kv, dim = rng.choice(((20, 4, 128), (24, 4, 256), (48, 8, 128), (32, 8, 128), (16, 2, 64), (8, 1, 256), (10, 10, 128)))
    dtype = rng.choice(("bf16", "fp16"))
    case = {"kind": kind, "heads": heads, "kv": kv, "dim": dim, "page": rng.choice((16, 32, 64, 128)), "cache": rng.choice(("e4m3", "e4m3", dtype)), "dtype": dtype}
    if kind == "append":
        context = _log(rng, 1, 8192)
        fresh = rng.choice((1, _log(rng, 1, context)))
        batch = _log(rng, 1, max(1, min(256, 2 ** 29 // (context * kv * dim), 2 ** 15 // fresh)))
        return case | {"batch": batch, "context": context, "fresh": fresh, "rot": rng.choice((dim, dim // 2, dim // 4)), "norm": rng.random() < 0.5}
    context = _log(rng, 1, 32768)
    fresh = rng.choice((1, 1, _log(rng, 1, min(context, 400))))
    batch = _log(rng, 1, max(1, min(128, 2 ** 28 // (context * kv * dim), 2 ** 28 // (context * heads * fresh))))
    return case | {"batch": batch, "context": context, "fresh": fresh, "window": rng.choice((0, 0, 0, 512))}


# ---- inputs ----------------------------------------------------------------------------------------------------
class _Draws:
    """Random tensors of one seed, on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, *shape, dtype=F32):
        return torch.empty(shape, dtype=F32, device=DEV).normal_(generator=self.gen).to(dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.empty(shape, dtype=F32, device=DEV).uniform_(lo, hi, generator=self.gen)

    def whole(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, device=DEV, generator=self.gen)


def _fresh(case):
    """New tokens of each sequence: ragged from ``fresh`` down to half of it."""
    return [max(1, case["fresh"] - b * 131 % (case["fresh"] // 2 + 1)) for b in range(case["batch"])]


def _lengths(case):
    """Tokens of each sequence: ragged from ``context`` down to half of it."""
    return [max(n, case["context"] - b * 977 % (case["context"] // 2 + 1)) for b, n in enumerate(_fresh(case))]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _table(case, r):
    """Every sequence's pages anywhere in the cache, a few of which are free."""
    needed = [-(-n // case["page"]) for n in _lengths(case)]
    order = torch.randperm(sum(needed) + 3, device=DEV, generator=r.gen).int()
    table = torch.full((len(needed), max(needed)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(needed):
        table[b, :n] = order[at:at + n]
        at += n
    return table, len(order)


def _exponent(amax):
    """The smallest e with amax / 2^e <= LARGEST."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x - 9 + (m > 0.875).int(), LEAST).clamp_min(LEAST)


def _power(e):
    return torch.ldexp(torch.ones_like(e, dtype=F32), e)


def _ragged(case):
    n = _fresh(case)
    starts = [0]
    for x in n:
        starts.append(starts[-1] + x)
    return (None if case["fresh"] == 1 else _ints(starts)), starts[-1]


def _append_inputs(case, seed):
    r, H, G, D, t = _Draws(seed), case["heads"], case["kv"], case["dim"], TYPES[case["dtype"]]
    table, pages = _table(case, r)
    starts, rows = _ragged(case)
    # the projection's rows: queries, keys and values beside each other
    qkv = r.normal(rows, (H + 2 * G) * D, dtype=t)
    shape = (pages, G, case["page"], D)
    s = {"kind": "append", "table": table, "lengths": _ints(_lengths(case)), "starts": starts, "k_scale": None, "v_scale": None,
         "q": qkv[:, :H * D].unflatten(1, (H, D)), "k_new": qkv[:, H * D:(H + G) * D].unflatten(1, (G, D)), "v_new": qkv[:, (H + G) * D:].unflatten(1, (G, D))}
    if case["cache"] == "e4m3":
        for name in ("k", "v"):
            s[name] = (r.normal(*shape) * 80).clamp_(-LARGEST, LARGEST).to(TYPES["e4m3"])
            s[name + "_scale"] = _power(r.whole(-8, -5, pages, G))
    else:
        s["k"], s["v"] = r.normal(*shape, dtype=t), r.normal(*shape, dtype=t)
    half = case["rot"] // 2
    angles = torch.arange(case["context"], device=DEV, dtype=F64)[:, None] * 10000.0 ** -(torch.arange(half, device=DEV, dtype=F64) / half)
    s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
    for name in ("q_weight", "k_weight"):
        s[name] = (1 + 0.1 * r.normal(D)).to(t) if case["norm"] else None
    return s


def _attend_inputs(case, seed):
    r, H, G, D, t = _Draws(seed), case["heads"], case["kv"], case["dim"], TYPES[case["dtype"]]
    table, pages = _table(case, r)
    starts, rows = _ragged(case)
    spread = torch.exp(0.5 * r.normal(2, G, 1, D))           # some channels are larger than others
    s = {"kind": "attend", "table": table, "lengths": _ints(_lengths(case)), "starts": starts, "window": case["window"] or None, "k_scale": None, "v_scale": None,
         "q": (1.5 * r.normal(rows, H, D) / spread[0].repeat_interleave(H // G, 0)[:, 0]).to(t)}
    for i, name in enumerate(("k", "v")):
        x = r.normal(pages, G, case["page"], D) * spread[i]
        if case["cache"] == "e4m3":
            scale = _power(_exponent(x.abs().amax((2, 3))))
            s[name], s[name + "_scale"] = (x / scale[:, :, None, None]).to(TYPES["e4m3"]), scale
        else:
            s[name] = x.to(t)
    return s


def _sample_inputs(case, seed):
    r, B, V = _Draws(seed), case["rows"], case["vocab"]
    logits = 2.0 * r.normal(B, V)
    likely = r.whole(0, V, B, 40)                        # a few tokens stand out, as after training
    logits.scatter_add_(1, likely, r.uniform(B, 40, lo=0.0, hi=10.0))
    s = {"kind": "sample", "logits": logits.to(TYPES[case["dtype"]]), "draws": r.uniform(B), "temperature": 1.0, "top_k": None, "top_p": 1.0, "min_p": 0.0}
    if case["filter"] == "mixed":
        pick = lambda *values, dtype=F32: torch.tensor(values, dtype=dtype, device=DEV)[r.whole(0, len(values), B)]
        s |= {"temperature": pick(0.0, 0.6, 0.8, 1.0, 1.3), "top_k": pick(0, 1, 20, 50, 1000, dtype=torch.int32), "top_p": pick(1.0, 0.8, 0.9, 0.95),
              "min_p": pick(0.0, 0.0, 0.02, 0.1)}
    elif case["filter"] == "k50p":
        s |= {"temperature": 0.7, "top_k": 50, "top_p": 0.9}
    elif case["filter"] == "p":
        s |= {"top_p": 0.95}
    elif case["filter"] == "min":
        s |= {"temperature": 1.2, "min_p": 0.05}
    return s


INPUTS = {"append": _append_inputs, "attend": _attend_inputs, "sample": _sample_inputs}


def prepare(case, seed):
    return INPUTS[case["kind"]](case, seed)


# ---- the operators -----------------------------------------------------------------------------------------------
def run(s):
    kind = s["kind"]
    if kind == "sample":
        if own:
            from tyr_b200.ops.sampling import sample
            return sample(s["logits"], s["draws"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return _sample(s)
    if own:
        from tyr_b200.ops.paged_cache import PagedStore, paged_append, paged_attention
        store = PagedStore(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if kind == "attend":
            return paged_attention(s["q"], store, s["table"], s["lengths"], s["starts"], window=s["window"])
        q = paged_append(store, s["k_new"], s["v_new"], s["table"], s["lengths"], s["starts"], q=s["q"], cos=s["cos"], sin=s["sin"],
                         q_weight=s["q_weight"], k_weight=s["k_weight"])
    elif kind == "attend":
        return _attend(s)
    else:
        q = _append(s)
    out = {"q": q, "k": s["k"], "v": s["v"]}
    return out if s["k_scale"] is None else out | {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _rows(s, rows):
    """(sequence, position, tokens before the call of each sequence) of the operands' rows."""
    B = s["lengths"].shape[0]
    starts = torch.arange(B + 1, device=DEV) if s["starts"] is None else s["starts"].long()
    row = torch.arange(rows, device=DEV)
    seq = torch.bucketize(row, starts[1:], right=True)
    held = s["lengths"].long() - (starts[1:] - starts[:-1])
    return seq, held[seq] + row - starts[seq], held


def _turned(x, weight, cos, sin, eps=1e-6):
    """Norm over the head, then rotation of the first channels, in pairs (i, i + half); 32 bits."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half:]], -1)


def _append(s):
    P = s["k"].shape[2]
    seq, pos, held = _rows(s, s["q"].shape[0])
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    page, slot = s["table"][seq, pos // P].long(), pos % P
    new = {"k": _turned(s["k_new"], s["k_weight"], cos, sin), "v": s["v_new"].float()}
    if s["k_scale"] is not None:
        begun = s["table"].gather(1, (held // P)[:, None])[:, 0].long()      # the pages that hold tokens of earlier calls
        begun_at = held % P
        old_slots = torch.arange(P, device=DEV) < begun_at[:, None]
    for name, x in new.items():
        store, scale = s[name], s[name + "_scale"]
        if scale is not None:
            amax = torch.full_like(scale, -1.0).scatter_reduce_(0, page[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
            want = torch.where(amax >= 0, _power(_exponent(amax)), scale)
            want[begun] = torch.where((begun_at > 0)[:, None], torch.maximum(want[begun], scale[begun]), want[begun])
            codes, factor = store[begun], (scale / want)[begun][:, :, None, None]
            moved = (codes.float() * factor).to(store.dtype)
            store[begun] = torch.where(old_slots[:, None, :, None], moved.view(torch.uint8), codes.view(torch.uint8)).view(store.dtype)
            scale.copy_(want)
            x = x / scale[page][:, :, None]
        store[page, :, slot] = x.to(store.dtype)
    return _turned(s["q"], s["q_weight"], cos, sin).to(s["q"].dtype)


def _attend(s):
    q, table, P, G = s["q"], s["table"].long().clamp_min(0), s["k"].shape[2], s["k"].shape[1]
    (T, H, D), B = q.shape, table.shape[0]
    seq, pos, held = _rows(s, T)
    at = pos - held[seq]                                    # place among the sequence's new tokens
    n = T if B == 1 else 1 if s["starts"] is None else int(at.max()) + 1

    def values(name):
        x = s[name][table].float()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][table][..., None, None]
        return x.transpose(1, 2).reshape(B, G, -1, D)
    rows = torch.zeros(B, n, H, D, device=DEV)
    rows[seq, at] = q.float()
    rows = rows.view(B, n, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, G, -1, D)
    x = (rows @ values("k").mT * D ** -0.5).view(B, G, n, H // G, -1)
    last, key = held[:, None] + torch.arange(n, device=DEV), torch.arange(x.shape[-1], device=DEV)
    seen = key <= last[..., None]
    if s["window"]:
        seen &= key > last[..., None] - s["window"]
    x = x.masked_fill_(~seen[:, None, :, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    o = (x.view(B, G, -1, x.shape[-1]) @ values("v")).view(B, G, n, H // G, D) / x.sum(-1, keepdim=True)
    return o.permute(0, 2, 1, 3, 4).reshape(B, n, H, D)[seq, at].to(q.dtype)


def _settings(s):
    """Temperature, top-k, top-p and min-p of each row, as a column in 64 bits."""
    B = s["logits"].shape[0]
    column = lambda v: (v.double() if torch.is_tensor(v) else torch.full((B,), float(v or 0), dtype=F64, device=DEV))[:, None]
    return column(s["temperature"]), column(s["top_k"]), column(s["top_p"]), column(s["min_p"])


def _sample(s):
    t, k, p, m = _settings(s)
    x, order = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)
    rank, x = torch.arange(x.shape[1], device=DEV), x.double()
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    before = w.cumsum(-1) - w
    kept = (w > 0) & (w >= m) & ((p >= 1) | (before < p * w.sum(-1, keepdim=True)) | (rank == 0))
    c = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0)).cumsum_(-1)
    token = (c <= s["draws"].double()[:, None] * c[:, -1:]).sum(-1)
    return torch.where(t[:, 0] > 0, token, order[:, 0])


# ---- the same in 64 bits -------------------------------------------------------------------------------------------
def _exact_turn(x, weight, cos, sin):
    x = x.to(F64)
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.to(F64)
    half = cos.shape[1]
    z = torch.complex(x[..., :half], x[..., half:2 * half]) * torch.complex(cos.to(F64), sin.to(F64))[:, None]
    return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)


def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    P, rows = case["page"], s["q"].shape[0]
    out = {"q": torch.empty(s["q"].shape, dtype=F64, device=DEV), "k": s["k"].to(F64), "v": s["v"].to(F64)}
    scales = {}
    if s["k_scale"] is not None:
        scales = {"k": s["k_scale"].to(F64), "v": s["v_scale"].to(F64)}
    table, at = s["table"].tolist(), 0
    for b, (n, length) in enumerate(zip(_fresh(case), _lengths(case))):
        first = length - n
        cos, sin = s["cos"][first:length], s["sin"][first:length]
        out["q"][at:at + n] = _exact_turn(s["q"][at:at + n], s["q_weight"], cos, sin)
        new = {"k": _exact_turn(s["k_new"][at:at + n], s["k_weight"], cos, sin), "v": s["v_new"][at:at + n].to(F64)}
        for j in range(first // P, (length - 1) // P + 1):
            lo, hi, page = max(first, j * P), min(length, (j + 1) * P), table[b][j]
            for name, x in new.items():
                x = x[lo - first:hi - first].transpose(0, 1)
                if scales:
                    unit = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)) / LARGEST)).clamp_min(LEAST))
                    if lo > j * P:
                        unit = torch.maximum(unit, scales[name][page])
                        out[name][page, :, :lo - j * P] *= (scales[name][page] / unit)[:, None, None]
                    scales[name][page] = unit
                    x = x / unit[:, None, None]
                out[name][page, :, lo - j * P:hi - j * P] = x
        at += n
    assert at == rows
    return out | {name + "_scale": unit for name, unit in scales.items()}


def _exact_attend(case, seed):
    if work(case)["flops"] > 4e11:
        return None
    s = _attend_inputs(case, seed)
    P, G, D, w = case["page"], case["kv"], case["dim"], case["window"]
    out, at = torch.empty(s["q"].shape, dtype=F64, device=DEV), 0
    for b, (n, length) in enumerate(zip(_fresh(case), _lengths(case))):
        pages = s["table"][b, :-(-length // P)].long()
        k, v = (s[name][pages].to(F64) * (1.0 if s[name + "_scale"] is None else s[name + "_scale"][pages].to(F64)[..., None, None]) for name in ("k", "v"))
        k, v = (x.transpose(0, 1).reshape(G, -1, D)[:, :length] for x in (k, v))
        q = s["q"][at:at + n].to(F64).unflatten(1, (G, -1))
        scores = torch.einsum("ngrd,gld->grnl", q, k) / math.sqrt(D)
        ago = torch.arange(length - n, length, device=DEV)[:, None] - torch.arange(length, device=DEV)
        scores = torch.where((ago >= 0) & (ago < w if w else ago >= 0), scores, -math.inf)
        out[at:at + n] = torch.einsum("grnl,gld->ngrd", scores.softmax(-1), v).flatten(1, 2)
        at += n
    return out


def _exact_sample(case, seed):
    s = _sample_inputs(case, seed)
    t, k, p, m = (x[:, 0].tolist() for x in _settings(s))
    tokens = []
    for b, row in enumerate(s["logits"].to(F64)):
        likely, order = torch.sort(row, dim=0, descending=True, stable=True)
        if t[b] <= 0:
            tokens.append(int(order[0]))
            continue
        if k[b] > 0:
            likely, order = likely[:int(k[b])], order[:int(k[b])]
        mass = torch.exp((likely - likely[0]) / t[b])
        ahead = torch.cat([mass.new_zeros(1), mass.cumsum(0)[:-1]])
        stays = mass >= m[b]
        if p[b] < 1:
            stays &= ahead < p[b] * mass.sum()
        stays[0] = True
        ids, back = order[stays].sort()
        line = mass[stays][back].cumsum(0)
        tokens.append(int(ids[min(int(torch.searchsorted(line, s["draws"][b].double() * line[-1], right=True)), len(ids) - 1)]))
    return torch.tensor(tokens, device=DEV)


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](case, seed)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * (vocab * TYPES[case["dtype"]].itemsize + 12), "flops": 2 * rows * vocab}
    H, G, D, wide, item = case["heads"], case["kv"], case["dim"], TYPES[case["dtype"]].itemsize, TYPES[case["cache"]].itemsize
    new, held = _fresh(case), _lengths(case)
    rows = sum(new)
    if case["kind"] == "append":
        pages = sum((n - 1) // case["page"] - (n - f) // case["page"] + 1 for f, n in zip(new, held))
        scales = 2 * 2 * 4 * pages * G if item == 1 else 0
        return {"bytes": rows * (2 * H * D * wide + 2 * G * D * (wide + item) + 4 * case["rot"]) + scales + 4 * pages, "flops": rows * (H + 2 * G) * D * 4}
    w = case["window"] or 2 ** 62
    keys = sum(min(n, w + f - 1) for f, n in zip(new, held))
    pairs = sum(min(p + 1, w) for f, n in zip(new, held) for p in range(n - f, n))
    return {"bytes": keys * 2 * G * D * item + 2 * rows * H * D * wide, "flops": 4 * pairs * H * D}
