"""The paged cache (ops/paged_cache.py): what is written and what attention reads, against plain 64-bit implementations of this file."""
import math

import pytest
import torch

from tyr_b200.ops import _common
from tyr_b200.ops import paged_cache as pc
from tyr_b200.ops.paged_cache import PagedStore, paged_append, paged_attention

F64 = torch.float64
FIELDS = ("k", "v", "k_scale", "v_scale")
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, torch.float8_e4m3fn: 2.0 ** -4}


class Batch:
    """Ragged sequences over scattered pages: ``held`` tokens in the cache before the call, ``new`` with it (None: one row each, none where 0)."""

    def __init__(self, held, new, G, P, D, dtype, cache, dev, seed=0, spare=2, rows_behind=0, strided=True, R=2, decode=False, heads=None):
        gen = torch.Generator().manual_seed(seed)
        self.held, self.new, self.G, self.P, self.D, self.H, self.dev = held, new, G, P, D, heads or G * R, dev
        self.lens = [h + n for h, n in zip(held, new)]
        need = [-(-n // P) for n in self.lens]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=gen)
        width = max(max(need), 1) + 1
        self.table = torch.full((len(held), width), 2 ** 30, dtype=torch.int32)         # what lies behind a sequence's pages is never looked at
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        if decode:
            assert all(n in (0, 1) for n in new)
            rows, self.row_of, starts = len(new), list(range(len(new))), None
            self.lens = [n if f else 0 for n, f in zip(self.lens, new)]
        else:
            rows, self.row_of, starts = self.starts[-1] + rows_behind, self.starts[:-1], torch.tensor(self.starts, dtype=torch.int32)
        self.rows = rows
        wide = torch.randn(rows, (self.H + 2 * G) * D + 8, generator=gen).to(dtype)
        cut = lambda a, n: wide[:, a * D:(a + n) * D].unflatten(1, (n, D))
        self.q, self.k, self.v = cut(0, self.H), cut(self.H, G), cut(self.H + G, G)
        if not strided:
            self.q, self.k, self.v = self.q.contiguous(), self.k.contiguous(), self.v.contiguous()
        # old tokens' numbers; the rest holds what an earlier owner or nobody left there
        x = torch.randn(2, pages, G, P, D, generator=gen)
        if cache == pc.E4M3:
            codes = (x * 90).clamp(-448, 448).to(cache)
            scales = torch.exp2(torch.randint(-9, -5, (2, pages, G), generator=gen).float())
            codes.view(torch.uint8)[:, order[at:]] = 0x7f
            scales[:, order[at:]] = math.nan
            for b, n in enumerate(self.lens):
                if n % P and need[b]:
                    codes.view(torch.uint8)[:, self.table[b, need[b] - 1], :, n % P:] = 0x7f
            self.store = PagedStore(codes[0].contiguous(), codes[1].contiguous(), scales[0].contiguous(), scales[1].contiguous())
        else:
            y = x.to(cache)
            y[:, order[at:]] = math.nan
            for b, n in enumerate(self.lens):
                if n % P and need[b]:
                    y[:, self.table[b, need[b] - 1], :, n % P:] = math.nan
            self.store = PagedStore(y[0].contiguous(), y[1].contiguous())
        to = lambda t: None if t is None else t.to(dev)
        self.q, self.k, self.v, self.table, starts = to(self.q), to(self.k), to(self.v), to(self.table), to(starts)
        self.args = (self.table, torch.tensor(self.lens, dtype=torch.int32, device=dev), starts)
        self.store = PagedStore(*(to(getattr(self.store, n)) for n in FIELDS))

    def copy(self):
        return PagedStore(*(None if getattr(self.store, n) is None else getattr(self.store, n).clone() for n in FIELDS))

    def sequence(self, b, store=None):
        """(keys, values) [G, length, D] of sequence b in 64 bits."""
        n = self.lens[b]
        pages = self.table[b, :-(-n // self.P)].long()
        k, v = (t.to(F64) for t in (store or self.store).values(pages))
        return tuple(t.transpose(0, 1).reshape(self.G, -1, self.D)[:, :n] for t in (k, v))


def oracle_attention(batch, window=None, scale=None):
    """(result, sum p |v|, largest sum of |q| |k| scale of a row) in 64 bits, rows of no sequence zero."""
    out = torch.zeros(batch.rows, batch.H, batch.D, dtype=F64, device=batch.dev)
    size, reach = torch.zeros_like(out), torch.zeros(batch.rows, batch.H, 1, dtype=F64, device=batch.dev)
    scale = batch.D ** -0.5 if scale is None else scale
    for b, n in enumerate(batch.lens):
        new, r0 = batch.new[b], batch.row_of[b]
        if not new or not n:
            continue
        k, v = batch.sequence(b)
        q = batch.q[r0:r0 + new].to(F64).unflatten(1, (batch.G, -1))
        s = torch.einsum("ngrd,gld->grnl", q, k) * scale
        pos = torch.arange(n - new, n, device=batch.dev)[:, None]
        key = torch.arange(n, device=batch.dev)
        s = s.masked_fill(~((key <= pos) & (key > pos - (window or n + 1))), -math.inf)
        p = s.softmax(-1)
        put = lambda t, x: t[r0:r0 + new].copy_(torch.einsum("grnl,gld->ngrd", p, x).flatten(1, 2))
        put(out, v), put(size, v.abs())
        reach[r0:r0 + new] = (torch.einsum("ngrd,gld->grnl", q.abs(), k.abs()).amax(-1) * abs(scale)).permute(2, 0, 1).flatten(1)[..., None]
    return out, size, reach


def check_attention(batch, got, window=None, scale=None, dtype=None):
    want, size, reach = oracle_attention(batch, window, scale)
    dtype = dtype or got.dtype
    # a probability is rounded to the products' type (f16 beside e4m3 and fp16 pages, else bf16); a score's sum of D products in fp32 is off by at most
    # (D + 3) roundings of the sum of magnitudes, and a probability's relative error is the scores' difference from the maximum's, twice that; exp2 and the sums
    # over the keys add some 2^-20
    p = HALF_STEP[torch.bfloat16 if batch.store.k.dtype == torch.bfloat16 else torch.float16]
    if got.is_cuda and gathered(batch):
        p = HALF_STEP[got.dtype]                       # the kernel on tcgen05 rounds them to the queries' type
    tol = HALF_STEP[dtype] * want.abs() + size * (1.01 * p + 2.0 ** -20 + 2 * 1.45 * (batch.D + 3) * 2.0 ** -24 * reach) + 1e-7
    err = (got.to(F64) - want).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} of the tolerance"


def oracle_rows(x, weight, cos, sin, pos, eps=1e-6, one_plus_w=False):
    x = x.to(F64)
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (weight.to(F64) + (1.0 if one_plus_w else 0.0))
    if cos is None:
        return x
    h, c, s = cos.shape[1], cos[pos].to(F64)[:, None], sin[pos].to(F64)[:, None]
    out = x.clone()
    out[..., :h] = x[..., :h] * c - x[..., h:2 * h] * s
    out[..., h:2 * h] = x[..., :h] * s + x[..., h:2 * h] * c
    return out


def check_append(batch, before, store, out, kw):
    """What the call left in ``store`` (``before``: a copy from before it) and returned."""
    q_want = torch.zeros(batch.rows, batch.H, batch.D, dtype=F64, device=batch.dev)
    q_size = torch.zeros_like(q_want)
    touched = torch.zeros(store.k.shape[:3], dtype=torch.bool, device=batch.dev)
    scaled = torch.zeros(store.k.shape[:1], dtype=torch.bool, device=batch.dev)
    P, f8 = batch.P, store.k_scale is not None
    for b, n in enumerate(batch.lens):
        new, r0 = batch.new[b], batch.row_of[b]
        if not new or not n:
            continue
        pos = torch.arange(n - new, n, device=batch.dev)
        rows = slice(r0, r0 + new)
        norm = dict(eps=kw.get("eps", 1e-6), one_plus_w=kw.get("one_plus_w", False))
        q_want[rows] = oracle_rows(batch.q[rows], kw.get("q_weight"), kw.get("cos"), kw.get("sin"), pos, **norm)
        q_size[rows] = oracle_rows(batch.q[rows].abs(), None if kw.get("q_weight") is None else kw["q_weight"].abs() + 2, None, None, pos).amax(-1, keepdim=True)
        for name, x in (("k", oracle_rows(batch.k[rows], kw.get("k_weight"), kw.get("cos"), kw.get("sin"), pos, **norm)), ("v", batch.v[rows].to(F64))):
            kept, old = getattr(store, name), getattr(before, name)
            # 32-bit arithmetic: the sum of squares, the root, three products and the rotation's sum, of the head's largest number
            near = 0.0 if name == "v" else (batch.D / 2 + 16) * 2.0 ** -24 * x.abs().amax(-1, keepdim=True)
            for j in range((n - new) // P, -(-n // P)):
                lo, hi, page = max(n - new, j * P), min(n, (j + 1) * P), int(batch.table[b, j])
                part, at = x[lo - n + new:hi - n + new].transpose(0, 1), slice(lo - j * P, hi - j * P)
                close = near if name == "v" else near[lo - n + new:hi - n + new].transpose(0, 1)
                got = kept[page, :, at].to(F64)
                touched[page, :, at] = True
                if not f8:
                    assert bool(((got - part).abs() <= HALF_STEP[kept.dtype] * part.abs() + close + 2.0 ** -25).all())
                    continue
                scaled[page] = True
                scale, was = getattr(store, name + "_scale")[page].to(F64), getattr(before, name + "_scale")[page].to(F64)
                want = torch.exp2(torch.ceil(torch.log2(part.abs().amax((1, 2)) / 448)).clamp_min(-100))
                if lo > j * P:
                    want = torch.maximum(want, was)
                assert torch.equal(scale, want), (scale, want)
                unit = scale[:, None, None]
                step = lambda y: torch.maximum(HALF_STEP[pc.E4M3] * y.abs(), torch.full_like(y, 2.0 ** -10))          # subnormals are 2^-9 apart
                assert bool(((got - part / unit).abs() <= step(part / unit) + 1.1 * close / unit).all())
                if lo > j * P:                                       # older tokens, in the new unit
                    held = old[page, :, :lo - j * P].to(F64) * (was / scale)[:, None, None]
                    assert bool(((kept[page, :, :lo - j * P].to(F64) - held).abs() <= torch.where(held.abs() < 2.0 ** -6, 2.0 ** -10, 0.0)).all())
                    touched[page, :, :lo - j * P] = True
    for name in ("k", "v"):
        raw = lambda s: getattr(s, name).view(torch.uint8 if f8 else torch.int16)
        assert torch.equal(raw(store)[~touched], raw(before)[~touched]), "a slot of no new token changed"
        if f8:
            a, b = getattr(store, name + "_scale"), getattr(before, name + "_scale")
            assert torch.equal(a[~scaled].view(torch.int32), b[~scaled].view(torch.int32)), "a scale of no new token changed"
    if out is not None:
        near = (batch.D / 2 + 16) * 2.0 ** -24 * q_size
        assert bool(((out.to(F64) - q_want).abs() <= HALF_STEP[out.dtype] * q_want.abs() + near + 2.0 ** -25).all())


def turns(positions, half, dev):
    ang = torch.arange(positions, dtype=F64)[:, None] * 10000.0 ** -(torch.arange(half, dtype=F64) / half)
    return dict(cos=ang.cos().float().to(dev), sin=ang.sin().float().to(dev))


RAGGED = dict(held=[0, 5, 63, 64, 0, 130, 17], new=[1, 3, 1, 1, 0, 70, 47])
STEPS = dict(held=[0, 15, 16, 200, 0, 64], new=[1, 1, 1, 1, 0, 1])

# (sequences, decode, G, R, P, D, type, cache, rotated half, norm)
APPENDS = [
    (STEPS, True, 4, 5, 16, 128, torch.bfloat16, pc.E4M3, 64, True),
    (STEPS, True, 2, 4, 64, 256, torch.float16, pc.E4M3, 32, True),
    (STEPS, True, 3, 1, 32, 64, torch.bfloat16, torch.bfloat16, 8, False),
    (STEPS, False, 2, 2, 128, 64, torch.bfloat16, pc.E4M3, 32, True),
    (RAGGED, False, 2, 3, 16, 128, torch.bfloat16, pc.E4M3, 64, True),
    (RAGGED, False, 1, 8, 32, 256, torch.float16, torch.float16, 32, True),
    (RAGGED, False, 4, 2, 64, 128, torch.float16, pc.E4M3, 16, False),
    (RAGGED, False, 2, 1, 128, 256, torch.bfloat16, pc.E4M3, 128, True),
    (RAGGED, False, 2, 2, 64, 64, torch.bfloat16, torch.bfloat16, None, True),
    (STEPS, True, 2, 3, 16, 128, torch.bfloat16, pc.E4M3, 12, True),
    (RAGGED, False, 2, 1, 32, 64, torch.float16, pc.E4M3, 20, True),
    (dict(held=[0], new=[1000]), False, 8, 6, 64, 128, torch.bfloat16, pc.E4M3, 64, False),
    (dict(held=[3] * 300, new=[n % 3 for n in range(300)]), False, 1, 2, 16, 64, torch.float16, pc.E4M3, 32, True),
]


def run_append(dev, seqs, decode, G, R, P, D, dtype, cache, half, norm, rows_behind=0, **more):
    batch = Batch(**seqs, G=G, R=R, P=P, D=D, dtype=dtype, cache=cache, dev=dev, decode=decode, rows_behind=rows_behind)
    kw = dict(more) if half is None else turns(max(batch.lens), half, dev) | more
    if norm:
        gen = torch.Generator().manual_seed(9)
        kw |= {n: (1 + 0.2 * torch.randn(D, generator=gen)).to(dtype).to(dev) for n in ("q_weight", "k_weight")}
    before = batch.copy()
    out = paged_append(batch.store, batch.k, batch.v, *batch.args, q=batch.q, **kw)
    check_append(batch, before, batch.store, out, kw)
    return batch


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_cpu(case):
    run_append("cpu", *APPENDS[case], rows_behind=0 if APPENDS[case][1] else 2)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_gpu(case):
    run_append("cuda", *APPENDS[case], rows_behind=0 if APPENDS[case][1] else 3)
    _common.raise_on_device_error()


def grow(dev, decode):
    """Three tokens of a page, each larger than those before."""
    G, P, D = 2, 16, 64
    store = PagedStore.allocate(3, G, P, D, dev)
    table = torch.tensor([[2]], dtype=torch.int32, device=dev)
    sizes, rows = (1.0, 0.01, 40.0, 3.0e4), []
    for i, size in enumerate(sizes):
        x = torch.randn(1, G, D, generator=torch.Generator().manual_seed(i)).clamp(-3, 3).mul(size).bfloat16().to(dev)
        rows.append(x)
        starts = None if decode else torch.tensor([0, 1], dtype=torch.int32, device=dev)
        assert paged_append(store, x, 2 * x, table, torch.tensor([i + 1], dtype=torch.int32, device=dev), starts) is None
    k, v = store.values(torch.tensor([2], device=dev))
    want = torch.stack([r[0] for r in rows], 1).double()
    scale = torch.exp2(torch.ceil(torch.log2(want.abs().amax((1, 2)) / 448)))
    assert torch.equal(store.k_scale[2].double(), scale) and torch.equal(store.v_scale[2].double(), 2 * scale)
    # two roundings: in the unit of the token's time, and to the final one's subnormals
    tol = HALF_STEP[pc.E4M3] * want.abs() * 1.07 + scale[:, None, None] * 2.0 ** -10 * 1.01
    assert bool(((k[0, :, :4].double() - want).abs() <= tol).all())
    assert bool(((v[0, :, :4].double() - 2 * want).abs() <= 2 * tol).all())
    assert torch.equal(store.k_scale[:2], torch.full_like(store.k_scale[:2], 2.0 ** -100))


def broken(dev, decode):
    """A number that is not finite marks its (page, head), until the page starts anew; extremes of size are held."""
    G, P, D = 2, 16, 64
    store = PagedStore.allocate(2, G, P, D, dev)
    table = torch.tensor([[1]], dtype=torch.int32, device=dev)

    def put(n, x):
        starts = None if decode else torch.tensor([0, 1], dtype=torch.int32, device=dev)
        paged_append(store, x, x, table, torch.tensor([n], dtype=torch.int32, device=dev), starts)
    x = torch.ones(1, G, D, dtype=torch.bfloat16, device=dev)
    put(1, x)
    for bad in (math.inf, -math.inf, math.nan):
        y = x.clone()
        y[0, 1, 5] = bad
        put(2, y)
        assert float(store.k_scale[1, 0]) == 2.0 ** -8 and math.isnan(store.k_scale[1, 1]) and math.isnan(store.v_scale[1, 1])
        assert not store.k[1, 1, 1].float().any() and not store.v[1, 1, 1].float().any()      # codes are numbers always
        put(3, x)
        assert math.isnan(store.k_scale[1, 1]) and float(store.v_scale[1, 0]) == 2.0 ** -8
        put(1, x)
        assert torch.equal(store.k_scale[1], torch.full_like(store.k_scale[1], 2.0 ** -8))
    for value, scale in ((0.0, 2.0 ** -100), (1e-39, 2.0 ** -100), (3.38e38, 2.0 ** 120), (448.0, 1.0), (450.0, 2.0)):
        put(1, x * value)
        assert torch.equal(store.k_scale[1], torch.full_like(store.k_scale[1], scale)), value
        got = store.k[1, :, 0].to(F64) * scale                   # 256 * 2^120 is beyond 32 bits
        want = (x * value)[0].double()
        assert bool(((got - want).abs() <= HALF_STEP[pc.E4M3] * want + scale * 2.0 ** -10).all())


@pytest.mark.parametrize("decode", (True, False))
def test_pages_grow_and_break_cpu(decode):
    grow("cpu", decode), broken("cpu", decode)


@pytest.mark.gpu
@pytest.mark.parametrize("decode", (True, False))
def test_pages_grow_and_break_gpu(decode):
    grow("cuda", decode), broken("cuda", decode)


# (sequences, decode, G, R, P, D, type, cache, window)
LONG = dict(held=[2999, 0, 700, 64, 0, 1, 4095], new=[1, 0, 1, 1, 1, 1, 1])
ATTENDS = [
    (STEPS, True, 4, 5, 16, 128, torch.bfloat16, pc.E4M3, None),
    (LONG, True, 2, 6, 32, 256, torch.bfloat16, pc.E4M3, None),
    (LONG, True, 2, 16, 64, 128, torch.float16, pc.E4M3, None),
    (LONG, True, 1, 40, 128, 128, torch.bfloat16, pc.E4M3, 100),
    (LONG, True, 2, 8, 16, 64, torch.float16, pc.E4M3, 700),
    (LONG, True, 3, 1, 64, 64, torch.bfloat16, torch.bfloat16, None),
    (LONG, True, 2, 5, 16, 128, torch.bfloat16, torch.bfloat16, 333),
    (LONG, True, 1, 12, 128, 256, torch.float16, torch.float16, None),
    (LONG, True, 2, 7, 32, 256, torch.bfloat16, torch.bfloat16, None),
    (RAGGED, False, 2, 3, 16, 128, torch.bfloat16, pc.E4M3, None),
    (RAGGED, False, 1, 8, 32, 256, torch.float16, torch.float16, None),
    (RAGGED, False, 2, 2, 64, 64, torch.bfloat16, pc.E4M3, 40),
    (RAGGED, False, 4, 1, 128, 128, torch.float16, pc.E4M3, 1),
    (RAGGED, False, 2, 4, 16, 64, torch.bfloat16, torch.bfloat16, 65),
    (dict(held=[900, 0, 3], new=[3, 2, 1]), False, 2, 2, 32, 128, torch.bfloat16, pc.E4M3, None),
    (dict(held=[1500, 0], new=[200, 333]), False, 2, 5, 16, 128, torch.bfloat16, torch.bfloat16, None),
    (dict(held=[1500, 0], new=[200, 333]), False, 1, 6, 64, 256, torch.bfloat16, pc.E4M3, 500),
    (dict(held=[7] * 150, new=[n % 3 for n in range(150)]), False, 1, 2, 16, 64, torch.float16, pc.E4M3, None),
    (dict(held=[0, 1000, 130, 7, 0, 300], new=[257, 1, 256, 0, 511, 129]), False, 2, 3, 16, 128, torch.bfloat16, pc.E4M3, None),
    (dict(held=[0, 1000, 130, 7, 0, 300], new=[257, 1, 256, 0, 511, 129]), False, 4, 4, 32, 64, torch.bfloat16, pc.E4M3, 100),
    (dict(held=[0, 1000, 130, 7, 0, 300], new=[257, 1, 256, 0, 511, 129]), False, 1, 5, 128, 128, torch.float16, torch.float16, 333),
    (dict(held=[0, 1000, 130, 7, 0, 300], new=[257, 1, 256, 0, 511, 129]), False, 2, 1, 64, 64, torch.bfloat16, torch.bfloat16, None),
    (dict(held=[0, 1000, 130, 7, 0, 300], new=[257, 1, 256, 0, 511, 129]), False, 1, 2, 64, 128, torch.float16, pc.E4M3, None),
    (dict(held=[5000], new=[1000]), False, 2, 4, 64, 128, torch.bfloat16, pc.E4M3, None),
    (dict(held=[40 * n for n in range(90)], new=[1] * 90), True, 2, 4, 64, 128, torch.bfloat16, pc.E4M3, None),
]


def gathered(batch):
    return batch.args[2] is not None and pc.gathers(batch.q.dtype, batch.store.k_scale is not None, batch.rows, len(batch.lens), batch.H, batch.G, batch.D,
                                                    batch.table.shape[1] * batch.P, 1.0)


def run_attention(dev, seqs, decode, G, R, P, D, dtype, cache, window, rows_behind=0):
    batch = Batch(**seqs, G=G, R=R, P=P, D=D, dtype=dtype, cache=cache, dev=dev, decode=decode, rows_behind=rows_behind, strided=False)
    batch.q = (batch.q * 2).contiguous()
    out = paged_attention(batch.q, batch.store, *batch.args, window=window)
    check_attention(batch, out, window)
    return batch


@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention_cpu(case):
    run_attention("cpu", *ATTENDS[case], rows_behind=0 if ATTENDS[case][1] else 2)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention_gpu(case):
    run_attention("cuda", *ATTENDS[case], rows_behind=0 if ATTENDS[case][1] else 3)
    _common.raise_on_device_error()


RAGGED_CASES = [i for i, c in enumerate(ATTENDS) if not c[1] and c[5] <= 128 and not (c[6] == torch.float16 and c[7] == pc.E4M3)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", RAGGED_CASES)
@pytest.mark.parametrize("way", (True, False))
def test_both_ways_over_ragged_rows(monkeypatch, case, way):
    monkeypatch.setattr(pc, "gathers", lambda *a: way)
    run_attention("cuda", *ATTENDS[case], rows_behind=3)
    _common.raise_on_device_error()


def test_way_by_rows_heads_and_types():
    bf, half = torch.bfloat16, torch.float16
    way = lambda rows, B=6, H=20, G=4, D=128, dtype=bf, f8=True, cap=3000, scale=0.1: pc.gathers(dtype, f8, rows, B, H, G, D, cap, scale)
    assert way(6 * 256) and way(6 * 100) and not way(6 * 8) and not way(6)
    assert not way(6 * 256, D=256) and not way(6 * 256, dtype=half) and way(6 * 256, dtype=half, f8=False) and not way(6 * 256, scale=-1.0)
    assert not way(6 * 256, cap=10 ** 6) and not way(2 * 64, B=2, H=10, G=10)


@pytest.mark.gpu
@pytest.mark.parametrize("R, P, D, cache", ((5, 16, 128, pc.E4M3), (6, 32, 256, pc.E4M3), (12, 64, 128, pc.E4M3), (8, 16, 64, pc.E4M3), (4, 32, 128, torch.bfloat16), (2, 128, 256, torch.bfloat16)))
def test_repeated_steps_agree(R, P, D, cache):
    """Whatever order the copies of a step's tiles arrive in: every one of many repetitions gives the same bits."""
    lens = [37 * n % 2900 + 1 for n in range(60)]
    batch = Batch(held=lens, new=[1] * 60, G=4, R=R, P=P, D=D, dtype=torch.bfloat16, cache=cache, dev="cuda", decode=True, strided=False)
    want = paged_attention(batch.q, batch.store, *batch.args)
    check_attention(batch, want)
    flush = torch.empty(2 ** 26, device="cuda")
    for i in range(150):
        if i % 5 == 0:
            flush.zero_()                                      # the pages come from memory again
        assert torch.equal(paged_attention(batch.q, batch.store, *batch.args), want)
    _common.raise_on_device_error()


@pytest.mark.gpu
@pytest.mark.parametrize("decode", (True, False))
def test_value_scales_of_any_spread(decode):
    """Values of one page 2^60 times another's, the large ones where the scores are least; and pages of nothing but zeros."""
    seqs = dict(held=[300, 100], new=[1, 1] if decode else [9, 20])
    batch = Batch(**seqs, G=2, R=4, P=16, D=128, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", decode=decode, strided=False)
    pages = batch.store.k.shape[0]
    batch.store.v_scale.copy_(torch.exp2(torch.arange(pages, device="cuda") % 7 * 20.0 - 70)[:, None].expand(-1, 2))
    batch.store.v_scale[::5] = 0.0
    batch.store.k_scale[1::3] = 2.0 ** -100
    want, size, reach = oracle_attention(batch)
    got = paged_attention(batch.q, batch.store, *batch.args)
    tol = HALF_STEP[torch.bfloat16] * want.abs() + size * (1.01 * 2.0 ** -11 + 2.0 ** -20 + 2.9 * 131 * 2.0 ** -24 * reach) + size.max() * 2.0 ** -60
    assert bool(((got.to(F64) - want).abs() <= tol).all())


@pytest.mark.gpu
def test_queries_of_any_size():
    for size in (1e-30, 1e-3, 1e3, 1e18):
        batch = Batch(held=[70, 3], new=[1, 1], G=2, R=4, P=16, D=128, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", decode=True, strided=False)
        batch.q = (batch.q * size).contiguous()
        scale = 0.1 / size
        check_attention(batch, paged_attention(batch.q, batch.store, *batch.args, scale=scale), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("way", (True, False))
def test_poisoned_pages_over_ragged_rows(monkeypatch, way):
    """Rows before a token that is no number do not show it, though they share its tile of keys."""
    monkeypatch.setattr(pc, "gathers", lambda *a: way)
    for name in ("k_scale", "v_scale"):
        batch = Batch(held=[100], new=[60], G=2, R=2, P=16, D=64, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", strided=False)
        getattr(batch.store, name)[int(batch.table[0, 8]), 1] = math.nan            # positions 128 to 143
        out = paged_attention(batch.q, batch.store, *batch.args)
        assert torch.isfinite(out[:, :2]).all() and torch.isfinite(out[:28]).all() and torch.isnan(out[28:, 2:]).all()


def poisoned(dev):
    """NaN in a page shows at the tokens that see it and at no others."""
    for name in ("k_scale", "v_scale"):
        batch = Batch(held=[100, 100], new=[1, 1], G=2, R=4, P=16, D=64, dtype=torch.bfloat16, cache=pc.E4M3, dev=dev, decode=True, strided=False)
        getattr(batch.store, name)[int(batch.table[1, 2]), 1] = math.nan
        out = paged_attention(batch.q, batch.store, *batch.args)
        assert torch.isfinite(out[0]).all() and torch.isfinite(out[1, :4]).all() and torch.isnan(out[1, 4:]).all()
        out = paged_attention(batch.q, batch.store, *batch.args, window=30)
        assert torch.isfinite(out).all()


def test_poisoned_pages_cpu():
    poisoned("cpu")


@pytest.mark.gpu
def test_poisoned_pages_gpu():
    poisoned("cuda")


def test_operands_reach_the_kernels_aligned():
    x = torch.arange(1 + 4 * 3 * 64, dtype=torch.bfloat16)[1:].view(4, 3, 64)
    assert x.data_ptr() % 16 and x.is_contiguous()
    for t in (x, x.transpose(0, 1), torch.arange(4 * 3 * 65, dtype=torch.bfloat16).view(4, 3, 65)[..., 1:], torch.arange(4 * 200, dtype=torch.bfloat16).view(4, 200)[:, 8:].unflatten(1, (3, 64))):
        y = pc._rows_of(t)
        assert torch.equal(y, t) and y.data_ptr() % 16 == 0 and y.stride(2) == 1 and all(s % 8 == 0 for s in y.stride()[:2])
    w = pc._aligned(x[0, 0], torch.bfloat16)
    assert torch.equal(w, x[0, 0]) and w.data_ptr() % 16 == 0
    assert pc._rows_of(y) is y


def small(dev="cpu", dtype=torch.bfloat16, cache=pc.E4M3, **kw):
    return Batch(held=[3, 20], new=[1, 1], G=2, R=2, P=16, D=64, dtype=dtype, cache=cache, dev=dev, decode=True, **kw)


def test_refusals_cpu():
    b = small()
    table, lens, _ = b.args
    ok = lambda **kw: paged_append(b.store, b.k, b.v, table, lens, **kw)
    t = turns(21, 16, "cpu")
    ok(q=b.q, **t)
    bad_page = table.clone()
    bad_page[0, 0] = b.store.k.shape[0]
    negative = table.clone()
    negative[1, 1] = -1
    for call in (
        lambda: ok(cos=t["cos"]), lambda: ok(cos=t["cos"][:20], sin=t["sin"][:20]), lambda: ok(q=b.q[:1]), lambda: ok(q=b.q.float()), lambda: ok(q_weight=torch.ones(63)),
        lambda: paged_append(b.store, b.k[:, :1], b.v[:, :1], table, lens), lambda: paged_append(b.store, b.k[..., :32], b.v[..., :32], table, lens),
        lambda: paged_append(b.store, b.k, b.v[:1], table, lens), lambda: paged_append(b.store, b.k[:1], b.v[:1], table, lens),
        lambda: paged_append(b.store, b.k, b.v, table.long(), lens), lambda: paged_append(b.store, b.k, b.v, table, lens.long()),
        lambda: paged_append(b.store, b.k, b.v, table[:1], lens), lambda: paged_append(b.store, b.k, b.v, table, lens, torch.tensor([0, 1], dtype=torch.int32)),
        lambda: paged_append(b.store, b.k, b.v, bad_page, lens), lambda: paged_append(b.store, b.k, b.v, negative, lens),
        lambda: paged_append(b.store, b.k, b.v, table, lens + 100), lambda: paged_append(b.store, b.k, b.v, table, lens, torch.tensor([0, 5, 2], dtype=torch.int32)),
        lambda: paged_append(b.store, b.k, b.v, table, lens, torch.tensor([0, 1, 3], dtype=torch.int32)),
        lambda: paged_attention(b.q[..., :32], b.store, table, lens), lambda: paged_attention(b.q[:, :3], b.store, table, lens), lambda: paged_attention(b.q[:1], b.store, table, lens),
        lambda: paged_attention(b.q, b.store, table, lens, window=0), lambda: paged_attention(b.q, b.store, bad_page, lens), lambda: paged_attention(b.q, b.store, table, lens + 100),
        lambda: PagedStore(b.store.k, b.store.v), lambda: PagedStore(b.store.k, b.store.v, b.store.k_scale), lambda: PagedStore(b.store.k, b.store.v, b.store.k_scale, b.store.v_scale.double()),
        lambda: PagedStore(b.store.k, b.store.v[:1], b.store.k_scale, b.store.v_scale), lambda: PagedStore(b.store.k.transpose(1, 2), b.store.v.transpose(1, 2), b.store.k_scale, b.store.v_scale),
        lambda: PagedStore(torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1, 16, 64, dtype=torch.int8)), lambda: PagedStore.allocate(0, 1, 16, 64, "cpu"),
    ):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_refusals_gpu():
    b = small("cuda")
    table, lens, _ = b.args
    cpu = small()
    odd = Batch(held=[3], new=[1], G=1, P=16, D=48, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", decode=True)
    page = Batch(held=[3], new=[1], G=1, P=8, D=64, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", decode=True)
    low = small("cuda", cache=torch.float16, dtype=torch.float16)
    for call in (
        lambda: paged_append(b.store, b.k.float(), b.v.float(), table, lens), lambda: paged_append(b.store, cpu.k, cpu.v, table, lens), lambda: paged_append(b.store, b.k, b.v, cpu.table, lens),
        lambda: paged_append(b.store, b.k, b.v, table, lens, **turns(30, 10, "cuda")), lambda: paged_append(b.store, b.k, b.v, table, lens, **turns(30, 16, "cpu")),
        lambda: paged_append(odd.store, odd.k, odd.v, *odd.args), lambda: paged_append(page.store, page.k, page.v, *page.args),
        lambda: paged_append(low.store, b.k, b.v, table, lens), lambda: paged_attention(b.q, low.store, table, lens), lambda: paged_attention(b.q.float(), b.store, table, lens),
        lambda: paged_attention(cpu.q, b.store, table, lens), lambda: paged_attention(odd.q, odd.store, *odd.args), lambda: paged_attention(page.q, page.store, *page.args),
    ):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_bad_tables_and_lengths_are_left_out_and_recorded():
    """The sequence that does not go together is recorded, its neighbour served; the kernels test every page and length before they use it."""
    for change in (lambda t, n, s: t[0].fill_(2 ** 30), lambda t, n, s: t[0].fill_(-5), lambda t, n, s: n[:1].fill_(10 ** 6), lambda t, n, s: s[:1].fill_(-1), lambda t, n, s: s[-1:].fill_(1000)):
        for decode in (True, False):
            b = Batch(held=[40, 20], new=[1, 1], G=2, R=2, P=16, D=64, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", decode=decode, strided=False)
            table, lens, starts = (None if t is None else t.clone() for t in b.args)
            moved = starts if starts is not None else torch.zeros(3, dtype=torch.int32, device="cuda")
            change(table, lens, moved)
            if decode and bool((moved != 0).any()):
                continue
            good = 0 if starts is not None and int(starts[-1]) == 1000 else 1
            out = paged_attention(b.q, b.store, table, lens, starts)
            with pytest.raises(RuntimeError):
                _common.raise_on_device_error()
            want = oracle_attention(b)[0]
            assert (out[good].double() - want[good]).abs().max() < 0.02 * want.abs().max()
            before = b.copy()
            q = paged_append(b.store, b.k, b.v, table, lens, starts, q=b.q)
            with pytest.raises(RuntimeError):
                _common.raise_on_device_error()
            assert torch.equal(q[good], b.q[good])
            page = int(b.table[good, (b.lens[good] - 1) // 16])
            assert not torch.equal(b.store.v[page].view(torch.uint8), before.v[page].view(torch.uint8))
            others = torch.arange(b.store.k.shape[0], device="cuda") != page
            assert torch.equal(b.store.v.view(torch.uint8)[others], before.v.view(torch.uint8)[others])


@pytest.mark.gpu
def test_views_streams_and_graphs():
    """Strided and misaligned operands, another stream, and two captured steps that are replayed at once over different batches."""
    b = Batch(held=[40, 500, 63], new=[1, 1, 1], G=2, R=4, P=32, D=128, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", decode=True)
    kw = turns(600, 64, "cuda")
    plain = b.copy()
    q = paged_append(plain, b.k.contiguous(), b.v.contiguous(), *b.args, q=b.q.contiguous(), **kw)
    o = paged_attention(q, plain, *b.args)
    shifted = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    wide_table = torch.full((3, b.table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide_table[:, :b.table.shape[1]] = b.table
    side = torch.cuda.Stream()
    for form in (lambda t: t, shifted, turned):
        store = b.copy()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            q2 = paged_append(store, form(b.k), form(b.v), wide_table[:, :b.table.shape[1]], b.args[1], q=form(b.q), **kw)
            o2 = paged_attention(form(q2), store, wide_table[:, :b.table.shape[1]], b.args[1])
        side.synchronize()
        assert torch.equal(q, q2) and torch.equal(o, o2) and torch.equal(store.k.view(torch.uint8), plain.k.view(torch.uint8)) and torch.equal(store.v_scale.view(torch.int32), plain.v_scale.view(torch.int32))

    c = Batch(held=[900, 10, 333], new=[1, 1, 1], G=2, R=4, P=32, D=128, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", decode=True, seed=5)
    kw = turns(1000, 64, "cuda")
    want, graphs = [], []
    for x in (b, c):
        store = x.copy()
        want.append(paged_attention(paged_append(store, x.k, x.v, *x.args, q=x.q, **kw), store, *x.args))
    torch.cuda.synchronize()
    for x in (b, c):
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = paged_attention(paged_append(x.store, x.k, x.v, *x.args, q=x.q, **kw), x.store, *x.args)
        graphs.append((graph, stream, out))
    for _ in range(20):
        for graph, stream, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, out), w in zip(graphs, want):
            assert torch.equal(out, w)
    _common.raise_on_device_error()


@pytest.mark.gpu
@pytest.mark.parametrize("cache", (pc.E4M3, torch.bfloat16))
def test_prompt_pieces_and_steps_together(cache):
    """Three sequences grow by pieces of prompts and by tokens, through both operators; every attention result against 64 bits over all that was given so far."""
    G, R, P, D, dev, dtype = 2, 4, 16, 128, "cuda", torch.bfloat16
    gen = torch.Generator(device=dev).manual_seed(3)
    store = PagedStore.allocate(40, G, P, D, dev, cache)
    order = torch.randperm(40, device=dev, generator=gen).int()
    table = torch.stack([order[:12], order[12:24], order[24:36]])
    kw = turns(200, 64, dev) | {"q_weight": torch.ones(D, dtype=dtype, device=dev), "k_weight": torch.ones(D, dtype=dtype, device=dev)}
    lens, kept = [0, 0, 0], [[], [], []]
    for new in ([33, 0, 7], [1, 1, 1], [16, 90, 0], [1, 1, 1], [1, 0, 1], [60, 3, 20], [1, 1, 1]):
        step = all(n < 2 for n in new)
        rows = 3 if step else sum(new)
        x = torch.randn(rows, (R + 2) * G * D, device=dev, generator=gen).to(dtype)
        q, k, v = x[:, :R * G * D].unflatten(1, (R * G, D)), x[:, R * G * D:(R + 1) * G * D].unflatten(1, (G, D)), x[:, (R + 1) * G * D:].unflatten(1, (G, D))
        lens = [n + m for n, m in zip(lens, new)]
        starts = [0, new[0], new[0] + new[1], sum(new)]
        first = [0, 1, 2] if step else starts[:3]
        lengths = torch.tensor([n if m or not step else 0 for n, m in zip(lens, new)], dtype=torch.int32, device=dev)
        args = (table, lengths, None if step else torch.tensor(starts, dtype=torch.int32, device=dev))
        out = paged_attention(paged_append(store, k, v, *args, q=q, **kw), store, *args)
        for b in range(3):
            if not new[b]:
                continue
            r = slice(first[b], first[b] + new[b])
            pos = torch.arange(lens[b] - new[b], lens[b], device=dev)
            kept[b].append((oracle_rows(k[r], kw["k_weight"], kw["cos"], kw["sin"], pos), v[r].to(F64)))
            keys, values = (torch.cat([y[i] for y in kept[b]]) for i in (0, 1))
            qs = oracle_rows(q[r], kw["q_weight"], kw["cos"], kw["sin"], pos)
            s = torch.einsum("ngrd,lgd->grnl", qs.unflatten(1, (G, R)), keys) / math.sqrt(D)
            s = s.masked_fill(torch.arange(lens[b], device=dev) > pos[:, None], -math.inf)
            p = s.softmax(-1)
            want = torch.einsum("grnl,lgd->ngrd", p, values).flatten(1, 2)
            size = torch.einsum("grnl,lgd->ngrd", p, values.abs()).flatten(1, 2)
            # the keys' roundings are independent, and so are the scores' errors: the root of the sum of (half a step, evenly spread: over sqrt 3) squares, of which six
            unit = HALF_STEP[cache]
            score = 6 * unit / math.sqrt(3) * torch.einsum("ngrd,lgd->grnl", qs.square().unflatten(1, (G, R)), keys.square()).sqrt().amax() / math.sqrt(D)
            tol = 2.0 ** -8 * want.abs() + size * (unit + 2.0 ** -8 + 2 * score)
            assert bool(((out[r].to(F64) - want).abs() <= tol).all())
        if step:
            assert all(bool((out[b] == 0).all()) for b in range(3) if not new[b])
    _common.raise_on_device_error()


SHIFTED = [(STEPS, True, 4, 5, 16, 128, torch.bfloat16, pc.E4M3, 64, True), (RAGGED, False, 2, 3, 32, 64, torch.float16, torch.float16, 16, True)]


@pytest.mark.parametrize("case", range(len(SHIFTED)))
def test_norm_of_one_plus_weight_cpu(case):
    run_append("cpu", *SHIFTED[case], one_plus_w=True, eps=0.03)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(SHIFTED)))
def test_norm_of_one_plus_weight_gpu(case):
    run_append("cuda", *SHIFTED[case], one_plus_w=True, eps=0.03)
    _common.raise_on_device_error()


def test_weights_of_another_type_and_gradients_are_refused():
    b = small()
    table, lens, _ = b.args
    weight = torch.ones(64)
    need = lambda t: t.clone().requires_grad_(True)
    for call in (lambda: paged_append(b.store, b.k, b.v, table, lens, k_weight=weight), lambda: paged_append(b.store, b.k, b.v, table, lens, q=b.q, q_weight=weight),
                 lambda: paged_append(b.store, need(b.k), b.v, table, lens), lambda: paged_append(b.store, b.k, need(b.v), table, lens),
                 lambda: paged_append(b.store, b.k, b.v, table, lens, q=need(b.q)), lambda: paged_attention(need(b.q), b.store, table, lens)):
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        paged_append(b.store, need(b.k), b.v, table, lens)
        paged_attention(need(b.q), b.store, table, lens)
    assert not b.store.k.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("cache", (pc.E4M3, torch.bfloat16))
def test_pages_behind_32_bits(monkeypatch, cache):
    """The same pages at the start of a small store and behind 2^32 elements of a large one: equal results."""
    G, P, D, far = 8, 128, 128, 32768                       # far * G * P * D = 2^32
    seqs = dict(held=[300, 0, 128, 1000], new=[1, 1, 1, 1])
    for decode, more in ((True, {}), (False, dict(held=[300, 0, 127, 1000], new=[70, 5, 1, 129]))):
        b = Batch(**(more or seqs), G=G, R=2, P=P, D=D, dtype=torch.bfloat16, cache=cache, dev="cuda", decode=decode)
        n, kw = b.store.k.shape[0], turns(1200, 64, "cuda")
        large = PagedStore.allocate(far + n, G, P, D, "cuda", cache)
        for name in FIELDS:
            if getattr(large, name) is not None:
                getattr(large, name)[far:] = getattr(b.store, name)
        table = torch.where(b.table < n, b.table + far, b.table)
        q = paged_append(b.store, b.k, b.v, *b.args, q=b.q, **kw)
        assert torch.equal(paged_append(large, b.k, b.v, table, *b.args[1:], q=b.q, **kw), q)
        for name in FIELDS:
            if getattr(large, name) is not None:
                raw = lambda t: t.view(torch.uint8)
                assert torch.equal(raw(getattr(large, name)[far:].contiguous()), raw(getattr(b.store, name)))
        for way in (False,) if decode else (False, True):
            monkeypatch.setattr(pc, "gathers", lambda *a: way)
            assert torch.equal(paged_attention(q, large, table, *b.args[1:]), paged_attention(q, b.store, *b.args))
        assert not large.k[:far].view(torch.uint8).any() and not large.v[:far].view(torch.uint8).any()
        del large
    _common.raise_on_device_error()


@pytest.mark.gpu
def test_two_streams_at_once(monkeypatch):
    """Different batches on two streams, both kernels of both ways in flight together: as one after the other."""
    batches = [Batch(held=[900, 40, 2000], new=[70, 33, 129], G=4, R=3, P=16, D=128, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", seed=s) for s in (1, 2)]
    steps = [Batch(held=[900, 40, 2000, 7], new=[1, 1, 1, 1], G=4, R=3, P=16, D=128, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", seed=s, decode=True) for s in (3, 4)]
    for way in (True, False):
        monkeypatch.setattr(pc, "gathers", lambda *a: way)
        want = [[paged_attention(b.q, b.store, *b.args) for b in pair] for pair in (batches, steps)]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
        for _ in range(5):
            for pair in (batches, steps):
                for s, b, g in zip(streams, pair, got):
                    with torch.cuda.stream(s):
                        g.append(paged_attention(b.q, b.store, *b.args))
        torch.cuda.synchronize()
        for i in (0, 1):
            for j, out in enumerate(got[i]):
                assert torch.equal(out, want[j % 2][i])
    _common.raise_on_device_error()


@pytest.mark.gpu
@pytest.mark.parametrize("way", ("step", False, True))
def test_rows_of_refused_sequences_are_zeros(monkeypatch, way):
    """A length beyond the table, more rows than tokens, rows outside the call's: recorded, zeros in the result, and the other sequences as without them."""
    monkeypatch.setattr(pc, "gathers", lambda *a: way is True)
    step = way == "step"
    b = Batch(held=[70, 300, 20], new=[1, 1, 1] if step else [40, 3, 60], G=2, R=2, P=16, D=64, dtype=torch.bfloat16, cache=torch.bfloat16, dev="cuda", decode=step, strided=False)
    table, lens, starts = b.args
    want = paged_attention(b.q, b.store, *b.args)
    long, few, first, last = lens.clone(), lens.clone(), None, None
    long[1] = 10 ** 6
    few[1] = 2
    cases = [(long, starts, 1)]
    if not step:
        first, last = starts.clone(), starts.clone()
        first[0], last[-1] = -1, 1000
        cases += [(few, starts, 1), (lens, first, 0), (lens, last, 2)]
    for n, s, bad in cases:
        for _ in range(3):
            torch.full_like(want, math.nan)                    # what the allocator hands out next
        out = paged_attention(b.q, b.store, table, n, s)
        rows = slice(bad, bad + 1) if step else slice(b.starts[bad], b.starts[bad + 1])
        with pytest.raises(RuntimeError):
            _common.raise_on_device_error()
        assert not out[rows].any()
        out[rows] = want[rows]
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("way", (False, True))
def test_a_length_just_beyond_the_table(monkeypatch, way):
    """Three pages of 16 hold 48 tokens, the laid out tile of keys 128: a length between them is refused like any other."""
    monkeypatch.setattr(pc, "gathers", lambda *a: way)
    b = Batch(held=[20, 8, 30], new=[10, 20, 1], G=2, R=2, P=16, D=64, dtype=torch.bfloat16, cache=torch.bfloat16, dev="cuda", strided=False)
    assert b.table.shape[1] == 3
    want = paged_attention(b.q, b.store, *b.args)
    for n in (49, 100, 128):
        lens = b.args[1].clone()
        lens[1] = n
        out = paged_attention(b.q, b.store, b.table, lens, b.args[2])
        with pytest.raises(RuntimeError):
            _common.raise_on_device_error()
        assert not out[10:30].any()
        out[10:30] = want[10:30]
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("way", ("step", False, True))
@pytest.mark.parametrize("P, D, dtype, cache", ((16, 64, torch.bfloat16, pc.E4M3), (64, 128, torch.bfloat16, torch.bfloat16), (16, 128, torch.float16, torch.float16), (128, 64, torch.bfloat16, torch.bfloat16),
                                                (32, 256, torch.bfloat16, pc.E4M3), (32, 256, torch.float16, torch.float16), (128, 128, torch.bfloat16, pc.E4M3)))
def test_pages_outside_the_cache_show_and_are_not_read(monkeypatch, way, P, D, dtype, cache):
    """The rows that see such a page are NaN, whatever the cache's first page holds; those before it, and other sequences, are as without it."""
    if way is True and D > 128:
        pytest.skip("heads of 256 have one way")
    monkeypatch.setattr(pc, "gathers", lambda *a: way is True)
    step = way == "step"
    b = Batch(held=[200, 600], new=[1, 1] if step else [500, 30], G=2, R=2, P=P, D=D, dtype=dtype, cache=cache, dev="cuda", decode=step, strided=False)
    want = paged_attention(b.q, b.store, *b.args)
    for at, page in ((1, 2 ** 31 - 1), (0, -1), (260 // P, -5), (260 // P, b.store.k.shape[0])):
        if step and at * P > 200:
            continue
        table = b.table.clone()
        table[0, at] = page
        out = paged_attention(b.q, b.store, table, *b.args[1:])
        with pytest.raises(RuntimeError):
            _common.raise_on_device_error()
        first, rows = max(0, at * P - 200), 1 if step else 500
        assert torch.isnan(out[first:rows]).all() and torch.equal(out[:first], want[:first]) and torch.equal(out[rows:], want[rows:])


def odd_values(dev, step, D, dtype, P=16, R=2):
    """Infinities and NaN among the values in 16 bits: in their channel, at the rows that see them, and nowhere else (a row before its neighbour's token, a window past it)."""
    b = Batch(held=[150, 70], new=[1, 1] if step else [300, 20], G=2, R=R, P=P, D=D, dtype=dtype, cache=dtype, dev=dev, decode=step, strided=False)
    b.q = (0.3 * b.q).contiguous()                         # no probability rounds to nothing
    clean = b.copy()
    places = ((0, 20, 0, 3, math.inf), (0, 90, 0, 11, math.nan), (0, 100, 1, D - 1, math.nan), (0, 145, 0, 9, -math.inf), (1, 66, 1, 17, math.inf)) if step else (
        (0, 20, 0, 3, math.inf), (0, 160, 0, 3, -math.inf), (0, 161, 1, D - 1, math.nan), (0, 299, 0, 40, math.inf), (0, 449, 0, 41, -math.inf), (1, 75, 1, 17, math.inf), (1, 89, 0, 0, math.nan))
    for s, key, g, d, value in places:
        page = int(b.table[s, key // P])
        clean.v[page, g, key % P, d], b.store.v[page, g, key % P, d] = 0.0, value
    for window in (None, 7, 60):
        want = paged_attention(b.q, clean, *b.args, window=window)
        assert torch.isfinite(want).all()
        for s, key, g, d, value in places:
            new, row0 = b.new[s], b.row_of[s]
            pos = torch.arange(b.lens[s] - new, b.lens[s])
            rows = row0 + torch.nonzero((pos >= key) & (pos < key + (window or 10 ** 6)))[:, 0]
            want[rows.to(dev), g * R:(g + 1) * R, d] += value
        out = paged_attention(b.q, b.store, *b.args, window=window)
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out.nan_to_num(0.0, 1e4, -1e4), want.nan_to_num(0.0, 1e4, -1e4))


@pytest.mark.parametrize("step", (True, False))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_odd_values_show_where_they_are_seen_cpu(step, dtype):
    odd_values("cpu", step, 64, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("step, R", ((True, 2), (True, 12), (False, 2), (False, 5)))
@pytest.mark.parametrize("D, P", ((64, 16), (128, 64), (256, 16), (128, 128)))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_odd_values_show_where_they_are_seen_gpu(monkeypatch, step, R, D, P, dtype):
    monkeypatch.setattr(pc, "gathers", lambda *a: False)
    odd_values("cuda", step, D, dtype, P, R)
    _common.raise_on_device_error()


@pytest.mark.gpu
@pytest.mark.parametrize("R", (2, 5))
@pytest.mark.parametrize("D, P", ((64, 16), (128, 64), (64, 128), (128, 16)))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_odd_values_show_where_they_are_seen_laid_out(monkeypatch, R, D, P, dtype):
    monkeypatch.setattr(pc, "gathers", lambda *a: True)
    odd_values("cuda", False, D, dtype, P, R)
    _common.raise_on_device_error()


@pytest.mark.gpu
@pytest.mark.parametrize("way", (True, False))
def test_values_in_8_bits_beyond_the_types_end(monkeypatch, way):
    """256 in units of 2^120 is infinite in 32 bits: rows that do not see it are as without it."""
    monkeypatch.setattr(pc, "gathers", lambda *a: way)
    b = Batch(held=[100], new=[300], G=2, R=2, P=16, D=64, dtype=torch.bfloat16, cache=pc.E4M3, dev="cuda", strided=False)
    b.store.v[int(b.table[0, 18]), 1] = 0.0                # positions 288 to 303
    want = paged_attention(b.q, b.store, *b.args)
    page = int(b.table[0, 18])
    b.store.v[page, 1, 5, 7] = 256.0
    b.store.v_scale[page, 1] = 2.0 ** 120
    out = paged_attention(b.q, b.store, *b.args)
    assert torch.equal(out[:188], want[:188]) and torch.equal(out[:, :2], want[:, :2]) and bool((out[193:, 2:, 7] > 1e30).all())


def test_gradients_of_norm_weights_and_rotations_are_refused():
    """A model's own parameters among them: the result would leave them without a gradient, and the CPU path would write a graph into the pages."""
    b = small()
    table, lens, _ = b.args
    need = lambda t: t.clone().requires_grad_(True)
    w, t = torch.ones(64, dtype=torch.bfloat16), turns(30, 16, "cpu")
    calls = (dict(k_weight=need(w)), dict(q=b.q, q_weight=need(w)), dict(cos=need(t["cos"]), sin=t["sin"]), dict(cos=t["cos"], sin=need(t["sin"])))
    for kw in calls:
        with pytest.raises(ValueError, match="no gradient"):
            paged_append(b.store, b.k, b.v, table, lens, **kw)
    with torch.no_grad():
        for kw in calls:
            paged_append(b.store, b.k, b.v, table, lens, **kw)
    assert not b.store.k.requires_grad
