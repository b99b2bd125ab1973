"""Draws of tokens (ops/sampling.py) against a row-by-row restatement in 64 bits; tokens are whole numbers and have to be equal."""
import math

import numpy as np
import pytest
import torch

from tyr_b200.models.generation import SamplingStrategy, sample_from_logits
from tyr_b200.ops.sampling import MAX_VOCAB, sample


def draw_of(row, u, t, k, p, m):
    """(token, how near the draw and the cuts come to another token, relative to the whole) of one row."""
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64)) + 0.0
    if not (x > -np.inf).any():
        return -1, 1.0
    if not t > 0:
        return int(np.flatnonzero(x == x.max())[0]), 1.0
    if (x == np.inf).any():
        x = np.where(x == np.inf, 0.0, -np.inf)
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    if k and k > 0:
        order = order[:k]
    w = np.exp((x[order] - x[order[0]]) / t)
    near = 1.0
    cum = np.concatenate([[0.0], np.cumsum(w)])
    stays = w >= min(m, 1.0)
    if p < 1:
        # equal weights make exact ties of whole multiples, which every way of summing them keeps
        gaps = np.abs(cum[:-1] - p * cum[-1]) / cum[-1]
        near = min(near, float(gaps[1:].min()) if len(w) > 1 and len(np.unique(w)) > 1 else 1.0)
        stays &= cum[:-1] < p * cum[-1]
    stays[0] = True
    ids = np.sort(order[stays])
    c = np.cumsum(np.exp((x[ids] - x[order[0]]) / t))
    near = min(near, float(np.abs(c[:-1] - u * c[-1]).min() / c[-1]) if len(c) > 1 and len(np.unique(x[ids])) > 1 else 1.0)
    past = np.flatnonzero(c > u * c[-1])
    return int(ids[past[0] if len(past) else -1]), near


def check(logits, draws, dev, **kw):
    """Equal tokens wherever nothing is nearer to a border than 1e-12 of the whole: the weights' relative error is 2e-13, and sums of 64-bit numbers add less."""
    B = logits.shape[0]
    got = sample(logits.to(dev), draws.to(dev), **{k: v.to(dev) if torch.is_tensor(v) else v for k, v in kw.items()})
    assert got.dtype == torch.int64 and got.shape == (B,)
    at = lambda name, b, default: default if kw.get(name) is None else (kw[name][b].item() if torch.is_tensor(kw[name]) else kw[name])
    rows, checked = logits.double().numpy(), 0
    for b in range(B):
        want, near = draw_of(rows[b], draws[b].item(), at("temperature", b, 1.0), at("top_k", b, 0), at("top_p", b, 1.0), at("min_p", b, 0.0))
        if near > 1e-12:
            checked += 1
            assert got[b].item() == want, (b, got[b].item(), want, near)
    assert checked >= B - 1 - B // 50
    return got


def mixed(B, gen):
    pick = lambda *v, dtype=torch.float32: torch.tensor(v, dtype=dtype)[torch.randint(0, len(v), (B,), generator=gen)]
    return dict(temperature=pick(0.0, 0.3, 0.8, 1.0, 1.7), top_k=pick(0, 1, 3, 50, 1000, 1500, 10 ** 6, dtype=torch.int32), top_p=pick(1.0, 0.0, 0.3, 0.9, 0.99), min_p=pick(0.0, 0.0, 0.02, 0.3, 1.0))


# (rows, vocabulary, type, spread of the logits, settings)
CASES = [
    (3, 1, torch.float32, 1.0, "mixed"), (5, 2, torch.bfloat16, 1.0, "mixed"), (33, 31, torch.float32, 2.0, "mixed"), (40, 500, torch.float16, 2.0, "mixed"),
    (64, 5003, torch.float32, 2.0, "mixed"), (64, 5003, torch.bfloat16, 4.0, "mixed"), (16, 50257, torch.float32, 2.0, "mixed"),
    (8, 50304, torch.float32, 2.0, dict()), (8, 50304, torch.float32, 0.0, dict(top_p=0.5)), (8, 20000, torch.float32, 0.0, dict(top_k=1500, top_p=0.9)),
    (8, 50304, torch.bfloat16, 0.3, dict(top_p=0.95)), (8, 33333, torch.float32, 1e-4, dict(top_p=0.95)), (8, 33333, torch.float32, 30.0, dict(top_p=0.999, temperature=2.0)),
    (8, 33333, torch.float32, 2.0, dict(top_k=5000, top_p=0.9)), (8, 33333, torch.float16, 2.0, dict(top_k=5000)), (8, 33333, torch.float32, 2.0, dict(top_k=1024, min_p=0.01)),
    (8, 33333, torch.float32, 2.0, dict(temperature=1e-3, top_p=0.9)), (8, 33333, torch.float32, 2.0, dict(temperature=50.0, top_p=0.7, top_k=20000)),
    (8, 33333, torch.float32, 2.0, dict(min_p=0.1)), (8, 33333, torch.float32, 2.0, dict(top_k=1)),
    (8, 33333, torch.bfloat16, 2.0, dict(top_k=1000, top_p=0.9)), (8, 33333, torch.bfloat16, 0.1, dict(top_k=300, top_p=0.5, min_p=0.9)), (8, 3001, torch.float16, 0.0, dict(top_k=1024, top_p=0.7)),
    (8, 1500, torch.float32, 0.0, dict(top_k=1024)), (8, 140, torch.float32, 2.0, dict(top_k=128, top_p=0.9)), (8, 33333, torch.float32, 60.0, dict(top_k=700, temperature=0.5)),
    (8, 33333, torch.float32, 1e-3, dict(top_k=1024, top_p=0.99, min_p=0.999)),
]
LARGE = [(3, 151936, torch.float32, 2.0, dict(temperature=0.7, top_k=50, top_p=0.9)), (150, 65536, torch.float32, 2.0, dict(top_p=0.95)), (20, 262144, torch.float32, 2.0, dict(top_p=0.95)),
         (5, 248320, torch.bfloat16, 2.0, "mixed"), (2, 300001, torch.float16, 3.0, dict(top_p=0.9)), (2, MAX_VOCAB, torch.float32, 2.0, dict(top_p=0.9, top_k=100000))]


def run(case, dev, seed=0):
    B, V, dtype, spread, kw = case
    gen = torch.Generator().manual_seed(seed)
    logits = (spread * torch.randn(B, V, generator=gen)).to(dtype)
    draws = torch.rand(B, generator=gen)
    check(logits, draws, dev, **(mixed(B, gen) if kw == "mixed" else kw))


@pytest.mark.parametrize("case", range(len(CASES)))
def test_draws_cpu(case):
    run(CASES[case], "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
def test_draws_gpu(case):
    for seed in range(3):
        run(CASES[case], "cuda", seed)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(LARGE)))
def test_draws_of_large_vocabularies(case):
    run(LARGE[case], "cuda")


def odd_rows(dev):
    V = 4000
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(14, V, generator=gen)
    x[0] = -math.inf                                      # nothing to choose from
    x[1] = math.nan
    x[2] = -math.inf
    x[2, 77] = -3.0                                       # one token is left
    x[3, 10], x[3, 500], x[3, 3999] = (math.inf,) * 3      # infinite ones share the draw
    x[4, ::2] = math.nan
    x[5, 1000:] = -math.inf
    x[6] = torch.finfo(torch.float32).min                  # a mask of the lowest value over everything
    x[7, 5:] = torch.finfo(torch.float32).min
    x[8] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)      # equal, whatever their sign
    x[9] = 3.4e38 * torch.sign(x[9])
    x[10, 3:] = 1e-42
    x[11, :] = torch.arange(V).flip(0).float() * 1e-3
    x[12, 20:] = -200.0
    x[13] = 1e-30 * x[13]
    draws = torch.tensor([0.5, 0.1, 0.9, 0.5, 0.3, 0.999, 0.25, 0.6, 0.75, 0.4, 0.2, 0.55, 0.99, 0.7])
    for kw in (dict(), dict(top_p=0.5), dict(top_k=3), dict(top_k=2000), dict(top_k=2000, top_p=0.5), dict(min_p=0.5), dict(temperature=0.0), dict(top_k=5, top_p=0.7, min_p=0.1, temperature=0.5)):
        got = check(x, draws, dev, **kw)
        assert got[0] == -1 and got[1] == -1 and got[2] == 77
    ends = torch.tensor([0.0, 1.0, 1.5, -1.0, math.nan])
    for kw in (dict(), dict(top_k=4), dict(top_p=0.9)):
        got = sample(torch.zeros(5, 8, device=dev), ends.to(dev), **kw).tolist()
        last = 3 if "top_k" in kw else 7
        assert got == [0, last, last, 0, last]
    assert sample(x.to(dev), draws.double().to(dev)).tolist() == sample(x.to(dev), draws.to(dev)).tolist()


def test_odd_rows_cpu():
    odd_rows("cpu")


@pytest.mark.gpu
def test_odd_rows_gpu():
    odd_rows("cuda")


@pytest.mark.gpu
def test_views_streams_and_graphs():
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide = 2 * torch.randn(6, 3 * 5003, device="cuda", generator=gen)
    draws = torch.rand(6, device="cuda", generator=gen)
    kw = dict(top_p=0.9, temperature=torch.full((6,), 0.9, device="cuda"))
    for view in (wide[:, 1:5004], wide[:, 4:5007], wide[:, ::3], wide[::2, :5003].repeat_interleave(2, 0), wide[:1, :5003].expand(6, -1)):
        want = sample(view.contiguous(), draws, **kw)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = sample(view, draws, **kw)
        side.synchronize()
        assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample(wide, draws, **kw)
    for _ in range(3):
        wide.normal_(generator=gen)
        draws.uniform_(generator=gen)
        graph.replay()
        assert torch.equal(out, sample(wide, draws, **kw))


def test_refusals():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    for call in (lambda: sample(x[0], u), lambda: sample(x[:, :0], u), lambda: sample(x, u[:1]), lambda: sample(x, u.long()), lambda: sample(x, u, temperature=-1.0), lambda: sample(x, u, top_p=math.nan),
                 lambda: sample(x, u, top_k=-1), lambda: sample(x, u, min_p=-0.1), lambda: sample(x, u, top_p=torch.ones(3)), lambda: sample(x, u, top_k=torch.ones(2)), lambda: sample(x.long(), u)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_refusals_gpu():
    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    for call in (lambda: sample(x, u.cpu()), lambda: sample(x.double(), u), lambda: sample(x, u, top_p=torch.ones(2)), lambda: sample(torch.zeros(1, MAX_VOCAB + 1, device="cuda"), u[:1])):
        with pytest.raises(ValueError):
            call()


def least_temperatures(dev):
    """Temperatures down to the least number that is none: the largest logits share the draw."""
    x = torch.tensor([[1.0, 3.0, 3.0, -2.0, math.nextafter(3.0, 0.0)], [0.0, 1e-45, 0.0, -1.0, 1e-45]])
    for t in (5e-324, 1e-310, 1e-300, 1e-60, torch.tensor([1e-45, 1e-45])):
        t = t.to(dev) if isinstance(t, torch.Tensor) else t
        for kw in (dict(), dict(top_k=4), dict(top_p=0.7), dict(min_p=0.5)):
            # 3.0 stands three times in fp32: thirds; 1e-45 twice, and at its own temperature zeros weigh 1 / e beside it: 0.37, 1.37, 1.74, 2.74
            for u, want in ((0.2, [1, 1]), (0.7, [4, 4])):
                assert sample(x.to(dev), torch.tensor([u, u], device=dev), temperature=t, **kw).tolist() == want


def test_least_temperatures_cpu():
    least_temperatures("cpu")


@pytest.mark.gpu
def test_least_temperatures_gpu():
    least_temperatures("cuda")


def test_top_k_is_a_whole_number():
    for k in (2.0, 2.5, "2"):
        with pytest.raises(ValueError):
            sample(torch.zeros(2, 8), torch.zeros(2), top_k=k)
    assert sample(torch.zeros(2, 8), torch.full((2,), 0.9), top_k=10 ** 12).tolist() == [7, 7]


@pytest.mark.gpu
def test_two_streams_at_once():
    rows = [3 * torch.randn(40, 50304, device="cuda", generator=torch.Generator(device="cuda").manual_seed(s)) for s in (1, 2)]
    draws = torch.rand(40, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    settings = (dict(top_p=0.9), dict(top_k=50, top_p=0.9), dict(), dict(top_k=2000))
    want = [[sample(x, draws, **kw) for kw in settings] for x in rows]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for kw in settings:
        for s, x, g in zip(streams, rows, got):
            with torch.cuda.stream(s):
                g.append(sample(x, draws, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))


@pytest.mark.gpu
@pytest.mark.parametrize("B, V, dtype", ((300, 20011, torch.float32), (230, 50304, torch.bfloat16), (70, 262144, torch.float16)))
def test_many_long_rows(B, V, dtype):
    """Rows that are read anew for every pass, against few at a time, which are held: the same tokens, odd rows among them."""
    gen = torch.Generator().manual_seed(V)
    x = (2 * torch.randn(B, V + 1, generator=gen)).to(dtype)[:, 1:]
    x[0], x[1, 5:], x[2, ::2], x[3, 7], x[4, V - 1] = -math.inf, -math.inf, math.nan, math.inf, math.inf
    x[4, 3], x[5], x[6, :V // 2] = math.inf, 0.25, -math.inf
    x, draws = x.cuda(), torch.rand(B, generator=gen).cuda()
    for kw in (dict(), dict(temperature=0.0), dict(top_p=0.9), dict(top_k=40, top_p=0.9), dict(top_k=1500), dict(top_k=3001, top_p=0.8), dict(min_p=0.02), dict(temperature=0.01, top_p=0.5)):
        got = sample(x, draws, **kw)
        held = torch.cat([sample(x[i:i + 10], draws[i:i + 10], **kw) for i in range(0, B, 10)])
        # cuts and draws within a rounding of the sums may fall otherwise: a part in 10^12 of the draws
        assert torch.equal(got, held)


def test_shared_memory_is_declared_as_it_is_accessed():
    """Dynamic shared memory follows a kernel's static part: without an alignment of its own, or a base that is rounded up, it starts where that ends."""
    import pathlib
    import re
    for unit in sorted((pathlib.Path(__file__).resolve().parents[1] / "csrc").glob("*.cu")):
        text = unit.read_text()
        for decl in re.findall(r"extern __shared__ [^;]*;", text):
            assert "__align__" in decl or " int " in decl or re.search(r"\+ 1023\)\s*&", text), (unit.name, decl)


def draws_of_zero(dev, B, V, dtype=torch.float32):
    """The first index that stays and weighs anything in 64 bits, however far below the largest: by its rank and weight, without sums."""
    gen = torch.Generator().manual_seed(V)
    x = 2 * torch.randn(B, V, generator=gen)
    x[:, :V // 8] -= 20.0                                   # unlikely ones come first
    x[::3, 3] = -200.0
    x[1::3, 0] = -math.inf
    x = x.to(dtype)
    zeros = torch.zeros(B)
    rows = x.double()
    order = torch.sort(rows, dim=1, descending=True, stable=True)[1]
    rank = torch.empty_like(order).scatter_(1, order, torch.arange(V).expand(B, -1))
    for kw in (dict(), dict(temperature=0.1), dict(temperature=0.02), dict(top_k=100, temperature=0.1), dict(top_k=1000, temperature=0.1), dict(top_k=V - 1, temperature=0.1),
               dict(top_p=0.9), dict(min_p=1e-30, temperature=0.2), dict(top_k=V - 2, top_p=0.99, min_p=1e-9, temperature=0.7), dict(top_k=900, min_p=1e-20, temperature=0.1)):
        w = torch.exp((rows - rows.amax(1, keepdim=True)) / kw.get("temperature", 1.0))
        first = torch.where(rank < kw.get("top_k", V), w, 0.0)
        by_rank = first.gather(1, order)
        before = torch.zeros_like(w).scatter_(1, order, by_rank.cumsum(1) - by_rank)
        stays = (first > 0) & (w >= kw.get("min_p", 0.0)) & ((before < kw.get("top_p", 2.0) * first.sum(1, keepdim=True)) | (rank == 0))
        want = stays.int().argmax(1)
        assert sample(x.to(dev), zeros.to(dev), **kw).tolist() == want.tolist(), kw


def test_draws_of_zero_cpu():
    draws_of_zero("cpu", 9, 5003)


@pytest.mark.gpu
@pytest.mark.parametrize("B, V, dtype", ((9, 5003, torch.float32), (4, 1500, torch.float16), (6, 151936, torch.bfloat16), (230, 50304, torch.float32)))
def test_draws_of_zero_gpu(B, V, dtype):
    draws_of_zero("cuda", B, V, dtype)


def greatest_temperatures(dev):
    """All finite logits weigh the same in the limit, though their distance is beyond 32 bits; -inf stays out."""
    V = 3000
    x = torch.where(torch.arange(V) % 2 == 0, 3.3e38, -3.3e38).repeat(3, 1)
    x[2, 1] = -math.inf
    order = torch.cat([torch.arange(0, V, 2), torch.arange(1, V, 2)])         # the larger ones first, then the others
    for t in (math.inf, 1e300, torch.full((3,), math.inf)):
        for kw in (dict(), dict(top_p=0.75), dict(top_k=2000), dict(top_k=800, top_p=0.5), dict(min_p=0.999)):
            stays = []
            for b in range(3):
                ids = order[~torch.isin(order, torch.tensor([1]))] if b == 2 else order
                ids = ids[:kw.get("top_k", V)]
                stays.append(sorted(ids[:math.ceil(kw.get("top_p", 1.0) * len(ids))].tolist()))
            u = torch.tensor([0.2505, 0.7505, 0.9005])
            want = [ids[math.floor(len(ids) * float(f))] for ids, f in zip(stays, u)]
            got = sample(x.to(dev), u.to(dev), temperature=t.to(dev) if torch.is_tensor(t) else t, **kw)
            assert got.tolist() == want, (t, kw)


def test_greatest_temperatures_cpu():
    greatest_temperatures("cpu")


@pytest.mark.gpu
def test_greatest_temperatures_gpu():
    greatest_temperatures("cuda")


def settings_of_no_number(dev):
    gen = torch.Generator().manual_seed(6)
    x, u = (2 * torch.randn(6, 4000, generator=gen)).to(dev), torch.rand(6, generator=gen).to(dev)
    nan, ones = torch.full((6,), math.nan, device=dev), torch.ones(6, device=dev)
    for kw in (dict(), dict(top_k=50), dict(top_k=2500), dict(temperature=0.5)):
        plain = sample(x, u, **kw)
        assert torch.equal(sample(x, u, min_p=nan, **kw), plain) and torch.equal(sample(x, u, top_p=nan, **kw), plain) and torch.equal(sample(x, u, min_p=-ones, **kw), plain)
    assert torch.equal(sample(x, u, temperature=nan), x.argmax(1)) and torch.equal(sample(x, u, min_p=3 * ones), x.argmax(1))


def test_settings_of_no_number_cpu():
    settings_of_no_number("cpu")


@pytest.mark.gpu
def test_settings_of_no_number_gpu():
    settings_of_no_number("cuda")
