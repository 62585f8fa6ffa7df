"""Sampling on the GPU against the definition in float64: whole numbers, so equal ones.

The inputs make the filters' borders matter (ties, integers, borders on a tie); where a border falls
between float64 values no result depends on the last bit of a sum: weights of equal logits are equal,
and random logits put the nearest border far from any sum's error."""
import math

import pytest
import torch

from dynakv_amd import _lib
from dynakv_amd.kernels.sampling import sample_tokens

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _one(x, u, t, k, p, mp):
    """The definition, for one row (float64 on the CPU)."""
    x = torch.where(torch.isnan(x), -math.inf, x)
    m = x.max()
    if m == -math.inf:
        return -1
    order = torch.sort(x, descending=True, stable=True).indices
    if not t > 0:
        return int(order[0])
    w = torch.where(x == m, 1.0, torch.exp((x - m) / t))
    w = torch.where(x == -math.inf, 0.0, w)
    if k > 0:
        order = order[:k]
    if p < 1:
        c = torch.cumsum(w[order], 0)
        order = order[:max(1, int((c - w[order] < p * c[-1]).sum()))]
    kept = order[w[order] >= mp]
    if len(kept) == 0:
        kept = order[:1]
    ids = torch.sort(kept).values
    c = torch.cumsum(w[ids], 0)
    i = int((c <= u * c[-1]).sum())
    if i >= len(ids):
        i = int((c < c[-1]).sum())
    return int(ids[i])


def _all(x, u, t, k, p, mp):
    at = lambda v, b: float(v[b]) if torch.is_tensor(v) else float(v)  # noqa: E731
    x, u = x.double().cpu(), u.double().cpu()
    t, p, mp = (v.cpu() if torch.is_tensor(v) else torch.tensor(v, dtype=torch.float32).item()
                for v in (t, p, mp))
    k = k.cpu() if torch.is_tensor(k) else k
    return [_one(x[b], float(u[b]), at(t, b), int(at(k, b)), at(p, b), at(mp, b))
            for b in range(x.shape[0])]


def _check(x, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    got = sample_tokens(x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    assert got.dtype == torch.int64 and got.shape == (x.shape[0],)
    want = _all(x, u, temperature, top_k, top_p, min_p)
    assert got.tolist() == want
    return got


def _inputs(dev, rows, V, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=g) * scale).to(DT[dtype])
    return x.to(dev), torch.rand(rows, generator=g).to(dev), g


SETTINGS = {
    "plain": {},
    "cold": dict(temperature=0.3),
    "hot": dict(temperature=5.0),
    "greedy": dict(temperature=0.0),
    "top_k": dict(top_k=40),
    "top_p": dict(top_p=0.9),
    "min_p": dict(min_p=0.05),
    "k_then_p": dict(top_k=100, top_p=0.8, temperature=0.7),
    "all": dict(top_k=300, top_p=0.95, min_p=0.02, temperature=1.3),
    "wide": dict(top_p=0.9999, top_k=100000),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("name", list(SETTINGS))
def test_settings(dev, name, dtype):
    print(f"[gpu] sample {name} {dtype}", flush=True)
    # short rows and many rows have a workgroup each, the others several
    for rows, V in ((9, 1000), (3, 32000), (2, 50257), (40, 20000), (150, 9001)):
        x, u, _ = _inputs(dev, rows, V, dtype, 7 * V + rows)
        _check(x, u, **SETTINGS[name])


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 7, 63, 64, 65, 511, 513, 1023, 1025, 8191, 131071, 131073,
                               200003, 524288])
def test_vocabulary_sizes(dev, V):
    print(f"[gpu] sample V={V}", flush=True)
    for dtype in ("bf16", "fp32"):
        x, u, _ = _inputs(dev, 2, V, dtype, V)
        _check(x, u, top_p=0.9)
        _check(x, u, top_k=3)
        _check(x, u)


@pytest.mark.gpu
def test_settings_of_each_row(dev):
    print("[gpu] sample per row", flush=True)
    x, u, g = _inputs(dev, 64, 5003, "fp32", 5)
    r = lambda lo, hi: (lo + (hi - lo) * torch.rand(64, generator=g)).to(dev)  # noqa: E731
    t, p, mp = r(0.0, 1.5), r(0.5, 1.1), r(-0.02, 0.1)
    t[::7] = 0.0
    t[1] = -1.0
    k = torch.randint(-1, 60, (64,), generator=g, dtype=torch.int32).to(dev)
    _check(x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    _check(x, u, temperature=t, top_k=5, top_p=p)
    _check(x, u, top_k=k, min_p=0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_ties(dev, dtype):
    """Few distinct logits: every border falls inside a run of equal ones, the lowest indices of
    which are kept; equal weights make a mass of exactly p or u a real case."""
    print(f"[gpu] sample ties {dtype}", flush=True)
    g = torch.Generator().manual_seed(9)
    x = torch.randint(-2, 3, (16, 4099), generator=g).to(DT[dtype]).to(dev)
    u = torch.rand(16, generator=g).to(dev)
    wide = torch.randint(-2, 3, (3, 60001), generator=g).to(DT[dtype]).to(dev)
    for kw in (dict(top_k=9000), dict(top_p=0.6), dict(top_k=40000, top_p=0.7), {}):
        _check(wide, u[:3], **kw)
    for kw in (dict(top_k=1), dict(top_k=2), dict(top_k=900), dict(top_k=4098), dict(top_p=0.5),
               dict(top_p=0.999), dict(top_k=1700, top_p=0.7), dict(min_p=1.0), dict(min_p=0.3),
               dict(top_p=1e-6), dict(temperature=0.0), {}):
        _check(x, u, **kw)
    same = torch.full((8, 1024), 0.5, dtype=DT[dtype], device=dev)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.9990234375, 0.125, 1 - 2.0**-24, 0.0009765625],
                     device=dev)
    assert _check(same, u).tolist() == [0, 256, 512, 768, 1023, 128, 1023, 1]
    assert _check(same, u, top_k=512).tolist() == [0, 128, 256, 384, 511, 64, 511, 0]
    assert _check(same, u, top_p=0.5).tolist() == [0, 128, 256, 384, 511, 64, 511, 0]
    zero = torch.zeros(2, 300, dtype=DT[dtype], device=dev)
    zero[:, ::2] = -0.0  # equal to 0: the order is the index's
    assert _check(zero, u[2:4], top_k=10).tolist() == [5, 7]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_what_cannot_be_taken(dev, dtype):
    print(f"[gpu] sample masked {dtype}", flush=True)
    inf, nan = math.inf, math.nan
    x, u, _ = _inputs(dev, 8, 3001, dtype, 21)
    low = torch.finfo(DT[dtype]).min
    x[0] = -inf                       # nothing to take
    x[1] = -inf
    x[1, 2222] = -3.0                 # one token
    x[2] = nan
    x[3] = nan
    x[3, 17] = 1.0
    x[4, 100] = inf                   # takes all the mass
    x[5, [5, 700, 3000]] = inf        # shared
    x[6] = low                        # the type's lowest value: an ordinary, equal logit
    x[7, ::2] = -inf
    x[7, 1::4] = nan
    for kw in ({}, dict(top_k=50), dict(top_p=0.8), dict(min_p=0.1, top_k=7, top_p=0.9),
               dict(temperature=0.0), dict(temperature=1e-30), dict(temperature=1e30, top_p=0.7)):
        got = _check(x, u, **kw).tolist()
        assert got[0] == -1 and got[1] == 2222 and got[2] == -1 and got[3] == 17 and got[4] == 100
        assert got[5] in (5, 700, 3000) and got[7] % 4 == 3


@pytest.mark.gpu
def test_extreme_settings(dev):
    print("[gpu] sample extreme settings", flush=True)
    x, u, _ = _inputs(dev, 6, 777, "fp32", 31)
    best = x.argmax(-1).tolist()
    for kw in (dict(top_p=0.0), dict(top_p=-1.0), dict(min_p=2.0), dict(top_k=1),
               dict(temperature=-1.0), dict(temperature=1e-38), dict(min_p=1.0)):
        assert _check(x, u, **kw).tolist() == best
    full = _check(x, u).tolist()
    for kw in (dict(top_p=1.0), dict(top_p=3.0), dict(top_k=777), dict(top_k=10**9),
               dict(top_k=-4), dict(min_p=0.0), dict(min_p=-1.0)):
        assert _check(x, u, **kw).tolist() == full
    # numbers that are no uniform ones stay inside what is kept
    odd = torch.tensor([1.0, 2.0, -1.0, math.nan, math.inf, 0.0], device=dev)
    got = sample_tokens(x, odd, top_k=5)
    for b in range(6):
        assert int(got[b]) in torch.topk(x[b], 5).indices.tolist()


@pytest.mark.gpu
def test_far_apart_logits(dev):
    """Borders far below the largest logit, and logits of both signs and all sizes."""
    print("[gpu] sample far apart", flush=True)
    g = torch.Generator().manual_seed(41)
    x = (torch.randn(6, 9001, generator=g) * torch.exp(6 * torch.randn(6, 9001, generator=g)))
    u = torch.rand(6, generator=g).to(dev)
    for dtype in ("fp32", "bf16"):
        y = x.clamp(-60000, 60000).to(DT[dtype]).to(dev)
        for kw in (dict(top_k=4500), dict(top_k=9000), dict(temperature=30000.0, top_p=0.6),
                   dict(temperature=1e4, top_k=5000, top_p=0.99)):
            _check(y, u, **kw)
        _check(y - 70000 if dtype == "fp32" else -y.abs(), u, top_k=4000, temperature=100.0)


@pytest.mark.gpu
def test_strides_and_out(dev):
    print("[gpu] sample strides", flush=True)
    for dtype in DT:
        whole, u, _ = _inputs(dev, 5, 4003, dtype, 51)
        x = whole[:, 3:3 + 3333]  # rows that start anywhere
        out = torch.full((5,), -9, dtype=torch.int64, device=dev)
        got = sample_tokens(x, u, top_p=0.9, out=out)
        assert got.data_ptr() == out.data_ptr()
        assert got.tolist() == _all(x, u, 1.0, 0, 0.9, 0.0)
    assert sample_tokens(whole[:0], u[:0]).shape == (0,)


@pytest.mark.gpu
def test_draws_follow_the_weights(dev):
    """A grid of u over [0, 1): every token is drawn on its share of the grid."""
    print("[gpu] sample shares", flush=True)
    n = 4096
    x = torch.tensor([0.0, 1.0, -1.0, 3.0, 2.0, -math.inf, 0.5], device=dev)
    u = (torch.arange(n, device=dev, dtype=torch.float32) + 0.5) / n
    got = sample_tokens(x.expand(n, -1).contiguous(), u, temperature=0.8)
    share = torch.bincount(got, minlength=7).double() / n
    want = torch.softmax(x.double() / torch.tensor(0.8, dtype=torch.float32).item(), 0)
    assert bool(((share - want).abs() <= 1.0 / n + 1e-9).all())
    assert bool((got[1:] >= got[:-1]).all())


@pytest.mark.gpu
def test_captured_and_repeated(dev):
    print("[gpu] sample graph", flush=True)
    x, u, g = _inputs(dev, 12, 32000, "bf16", 61)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        sample_tokens(x, u, top_k=50, top_p=0.9)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            got = sample_tokens(x, u, top_k=50, top_p=0.9)
    for _ in range(4):
        x.copy_((torch.randn(12, 32000, generator=g) * 3).to(torch.bfloat16))
        u.copy_(torch.rand(12, generator=g))
        gr.replay()
        torch.cuda.synchronize()
        assert got.tolist() == sample_tokens(x, u, top_k=50, top_p=0.9).tolist()
        assert got.tolist() == _all(x, u, 1.0, 50, 0.9, 0.0)


def _row(kind, V, g):
    x = torch.randn(V, generator=g)
    if kind == "tiny":            # all next to 0: 1 - 2^-30 and the like
        return x * 1e-7
    if kind == "near":            # some next to 0, beside zeros of both signs and ordinary ones
        x = x * 2
        x[::5], x[1::7], x[2::7] = x[::5] * 1e-5, 0.0, -0.0
        return x
    if kind == "near_below":      # those next to 0 are the largest
        return torch.where(x > 0.5, x * 1e-6, -x.abs() * 4)
    if kind == "zeros":           # half of them 0
        return torch.where(x > 0, 0.0, x * 3)
    if kind == "below":           # all far below 0
        return x * 3 - 300.0
    if kind == "above":
        return x * 2 + 1000.0
    if kind == "spread":          # more values than there are bins
        return torch.exp(x * 4) * x.sign()
    if kind == "masked":          # most of them at the type's lowest value, some -infinity
        return torch.where(x > 1.0, x * 2, torch.where(x > 0, -65504.0, -math.inf))
    if kind == "equal":
        return torch.full((V,), -3.25)
    if kind == "nan":             # of both signs
        x = x * 2.5
        x[::3], x[1::9] = math.nan, -math.nan
        return x
    if kind == "infinite":
        x[::11] = math.inf
        return x
    return x * 2.5


KINDS = ["tiny", "near", "near_below", "zeros", "below", "above", "spread", "masked", "equal", "nan",
         "infinite", "plain"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kind", KINDS)
def test_logits_of_every_kind(dev, kind, dtype):
    """Where 16-bit logits are counted by value: what lies next to 0, ranges with more values than
    bins, constants; each filter, cold and hot."""
    print(f"[gpu] sample logits {kind} {dtype}", flush=True)
    g = torch.Generator().manual_seed(61)
    for V in (777, 20000):
        x = torch.stack([_row(kind, V, g) for _ in range(6)]).to(DT[dtype]).to(dev)
        u = torch.rand(6, generator=g).to(dev)
        for t in (1.0, 0.05, 40.0):
            _check(x, u, temperature=t)
            _check(x, u, temperature=t, top_k=V // 3)
            _check(x, u, temperature=t, top_p=0.97)
            _check(x, u, temperature=t, top_p=0.5, top_k=V // 2, min_p=0.3)
        _check(x, u, top_k=V - 1, top_p=0.999999)
    # long rows in a workgroup each
    x = torch.stack([_row(kind, 90001, g) for _ in range(2)]).to(DT[dtype]).to(dev)
    x, u = x.repeat(70, 1), torch.rand(140, generator=g).to(dev)
    got = [sample_tokens(x, u, **kw).tolist() for kw in ({}, dict(top_p=0.9), dict(top_k=1000))]
    few = torch.cat([torch.arange(4), torch.arange(137, 140)])
    for kw, t in zip(((0, 1.0), (0, 0.9), (1000, 1.0)), got):
        p = torch.tensor(kw[1], dtype=torch.float32).item()
        want = _all(x[few.to(dev)], u[few.to(dev)], 1.0, kw[0], p, 0.0)
        assert [t[int(i)] for i in few] == want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_same_with_and_without_the_tensor_module(dev, dtype, monkeypatch):
    print(f"[gpu] sample without the tensor module {dtype}", flush=True)
    inputs = [_inputs(dev, rows, V, dtype, V) for rows, V in ((1, 1), (5, 999), (3, 131072), (0, 5))]

    def run():
        out = []
        for x, u, _ in inputs:
            n = x.shape[0]
            each = [torch.full((n,), v, device=dev) for v in (0.7, 0.8, 0.01)]
            k = torch.full((n,), 50, dtype=torch.int32, device=dev)
            out += [sample_tokens(x, u), sample_tokens(x, u, top_k=10**12),
                    sample_tokens(x, u, temperature=1, top_k=-3, top_p=0.9, min_p=0.1),
                    sample_tokens(x, u, temperature=each[0], top_k=k, top_p=each[1], min_p=each[2]),
                    sample_tokens(x[:, :max(1, x.shape[1] - 1)], u, top_k=7)]
        return out

    fast = run()
    monkeypatch.setattr(_lib, "_tensor_calls", None)
    for a, b in zip(run(), fast):
        assert a.dtype == b.dtype == torch.int64 and torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_borders_among_many_equal_logits(dev, dtype):
    """Thousands of equal logits at the border beside some next to them, of both signs: the search by
    digits, for top-k, top-p and both."""
    print(f"[gpu] sample many equal {dtype}", flush=True)
    g = torch.Generator().manual_seed(71)
    for V in (9001, 30000):
        x = torch.randn(5, V, generator=g) * 2.5
        x[torch.rand(5, V, generator=g) < 0.9] = 0.0
        x[1, ::13], x[2, ::17], x[3] = 1e-6, -1e-6, x[3] - 7.75
        x[4, ::3] = -0.0
        x = x.to(DT[dtype]).to(dev)
        u = torch.rand(5, generator=g).to(dev)
        for kw in (dict(top_p=0.9), dict(top_p=0.5), dict(top_k=V // 2), dict(top_k=V - 50),
                   dict(top_k=V // 2, top_p=0.8), dict(temperature=0.3, top_p=0.99, top_k=V // 3)):
            _check(x, u, **kw)
