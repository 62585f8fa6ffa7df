"""The paged cache's operators on the GPU against the formulas in float64.

Every pool starts full of NaN and every table ends in ids outside the pool, so a slot that is read
without having been written, or a page that is not the request's, shows in the result; every write
is checked by comparing the whole pool. Tolerances count the roundings (a 16-bit value is off by at
most half a step, eps / 2 relative): see ``_append_tol`` and ``_attend_tol``."""
import math
import threading

import pytest
import torch

from dynakv_amd import _lib
from dynakv_amd.kernels.paged import PagedBatch, PagedKVCache, paged_append, paged_attention

DH = 128
BF, FP = torch.bfloat16, torch.float16


class Step:
    """A step's batch and pools: ``new`` and ``lens`` per request, pages in random order."""

    def __init__(self, dev, new, lens, *, hkv=8, ps=16, dtype=BF, seed=0, layout="plain", pad=0,
                 spare=2, data=True):
        self.dev, self.new, self.lens, self.hkv, self.ps, self.dtype = dev, new, lens, hkv, ps, dtype
        g = self.g = torch.Generator().manual_seed(seed)
        need = [-(-n // ps) for n in lens]
        pages = sum(need) + spare
        ids = torch.randperm(pages, generator=g).tolist()
        cols = max(need) + 2
        self.table = torch.full((len(new), cols), pages + 7, dtype=torch.int32)  # not in the pool
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1]
        self.T = self.rows + pad
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        self.batch = PagedBatch(self.table.to(dev), i32(self.starts), i32(lens), rows=self.rows,
                                max_new=max(new), max_len=max(lens),
                                min_new=min([n for n in new if n], default=0))
        self.k = self.pool(pages, layout)
        self.v = self.pool(pages, layout)
        if data:  # the requests' tokens, the step's own included
            for b, n in enumerate(lens):
                for t0 in range(0, n, ps):
                    m = min(ps, n - t0)
                    page = int(self.table[b, t0 // ps])
                    for t in (self.k, self.v):
                        t[page, :, :m] = self.rand(hkv, m, DH)

    def pool(self, pages, layout):
        nan = float("nan")
        if layout == "plain":
            return torch.full((pages, self.hkv, self.ps, DH), nan, dtype=self.dtype, device=self.dev)
        # heads first, or pages with room between them
        if layout == "heads_first":
            return torch.full((self.hkv, pages, self.ps, DH), nan, dtype=self.dtype,
                              device=self.dev).transpose(0, 1)
        return torch.full((pages, self.hkv + 1, self.ps + 16, DH), nan, dtype=self.dtype,
                          device=self.dev)[:, :self.hkv, :self.ps]

    def rand(self, *dims, scale=1.0):
        return (torch.randn(*dims, generator=self.g) * scale).to(self.dtype).to(self.dev)

    def tokens(self, pool, b, g):
        """(len, 128) float64: the keys or values of request b, KV head g."""
        n = self.lens[b]
        ids = self.table[b, :-(-n // self.ps)].long().to(self.dev)
        return pool[ids, g].reshape(-1, DH)[:n].double()


# ---------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------
def _turn(y, pos, freq):
    """(n, heads, 128) rotated at positions (n,), all float64."""
    ang = pos[:, None, None] * freq
    a, b = y[..., :64], y[..., 64:]
    c, s = torch.cos(ang), torch.sin(ang)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _append_reference(s, qkv, heads, freq, q_norm=None, k_norm=None, eps=1e-6):
    """(queries, keys, values) of the step's rows in float64, and the sizes the tolerance uses."""
    x = qkv[:s.rows].double().reshape(s.rows, -1)[:, :(heads + 2 * s.hkv) * DH]
    x = x.view(s.rows, heads + 2 * s.hkv, DH)
    q, k, v = x[:, :heads], x[:, heads:heads + s.hkv], x[:, heads + s.hkv:]
    norm = lambda t, w: t if w is None else (  # noqa: E731
        t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * w.double())
    q, k = norm(q, q_norm), norm(k, k_norm)
    pos = torch.cat([torch.arange(n - m, n, dtype=torch.float64)
                     for m, n in zip(s.new, s.lens)]).to(s.dev)
    size = lambda t: (t[..., :64].abs() + t[..., 64:].abs()).repeat(1, 1, 2)  # noqa: E731
    return _turn(q, pos, freq), _turn(k, pos, freq), v, size(q), size(k)


def _append_tol(want, size, dtype):
    """Half a step of the result; before that fp32 work on the pair: the norm's sum of 128 squares,
    root, division and two products (a relative 2^-24 each, under 32 of them), the part of a
    revolution in fp32 (2 pi 2^-25) and the sine and cosine instructions (2^-18 at most is assumed
    of them), each times the pair's size."""
    return torch.finfo(dtype).eps / 2 * want.abs() + size * (2.0**-18 + 2.0**-19) + 1e-30


def _freq(dev, theta):
    return torch.tensor([theta ** (-2.0 * j / DH) for j in range(64)], dtype=torch.float64,
                        device=dev)


def _check_append(s, heads, *, theta=500000.0, norms=False, inv_freq=None, qkv=None, out=None,
                  wide=0):
    if qkv is None:
        qkv = s.rand(s.T, (heads + 2 * s.hkv) * DH + wide)
    qn = kn = None
    if norms:
        qn, kn = 1 + s.rand(DH, scale=0.2), 1 + s.rand(DH, scale=0.2)
    k0, v0, x0 = s.k.clone(), s.v.clone(), qkv.clone()
    q = paged_append(qkv, s.k, s.v, s.batch, heads=heads,
                     theta=None if inv_freq is not None else theta, inv_freq=inv_freq, q_norm=qn,
                     k_norm=kn, out=out)
    freq = (_freq(s.dev, theta) if inv_freq is None
            else torch.tensor(inv_freq, dtype=torch.float64, device=s.dev))
    wq, wk, wv, sq, sk = _append_reference(s, qkv, heads, freq, qn, kn)
    assert torch.equal(qkv, x0), "the projection was written to"
    assert bool(((q[:s.rows].double() - wq).abs() <= _append_tol(wq, sq, s.dtype)).all())
    # the pools: the written slots within their tolerance, every other slot as it was
    at = 0
    for b, (m, n) in enumerate(zip(s.new, s.lens)):
        for t in range(n - m, n):
            page, slot = int(s.table[b, t // s.ps]), t % s.ps
            err = (s.k[page, :, slot].double() - wk[at]).abs()
            assert bool((err <= _append_tol(wk[at], sk[at], s.dtype)).all()), (b, t)
            assert torch.equal(s.v[page, :, slot].double(), wv[at]), (b, t)
            k0[page, :, slot], v0[page, :, slot] = s.k[page, :, slot], s.v[page, :, slot]
            at += 1
    bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731  (NaN equals itself)
    assert torch.equal(bits(s.k), bits(k0)) and torch.equal(bits(s.v), bits(v0))
    return q


APPEND = {
    # name: (new tokens, lengths, query heads, KV heads, page, dtype, norms, layout)
    "one_token": ([1], [1], 4, 2, 16, BF, False, "plain"),
    "step_of_five": ([1] * 5, [33, 1, 16, 17, 250], 32, 8, 16, BF, False, "plain"),
    "prompts": ([40, 1, 65], [40, 1, 65], 8, 2, 32, FP, True, "plain"),
    "chunk_far_out": ([33], [100033], 4, 1, 128, FP, False, "plain"),
    "none_and_some": ([0, 3, 0, 0, 18, 0], [5, 3, 0, 31, 20, 7], 6, 3, 16, BF, True, "plain"),
    "heads_first": ([9, 2], [30, 50], 14, 2, 16, FP, True, "heads_first"),
    "pages_apart": ([9, 2], [30, 50], 8, 8, 64, BF, False, "apart"),
    "many_requests": ([1, 0, 2] * 70, [5, 9, 18] * 70, 2, 1, 16, BF, False, "plain"),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(APPEND))
def test_append(dev, name):
    new, lens, hq, hkv, ps, dt, norms, layout = APPEND[name]
    print(f"[gpu] paged append {name}", flush=True)
    s = Step(dev, new, lens, hkv=hkv, ps=ps, dtype=dt, layout=layout, seed=3, data=False)
    _check_append(s, hq, norms=norms)


@pytest.mark.gpu
def test_append_given_frequencies_and_strides(dev):
    print("[gpu] paged append frequencies, strides", flush=True)
    inv = [(1.0 if j < 20 else 0.125) * 10000.0 ** (-2.0 * j / DH) for j in range(64)]
    s = Step(dev, [7, 20], [4000, 20], hkv=2, dtype=FP, seed=4, data=False)
    whole = torch.full((s.T, 5, 2 * DH), 5.0, dtype=FP, device=dev)
    out = whole[:, 1:, :DH]  # rows and heads apart
    q = _check_append(s, 4, inv_freq=inv, out=out, wide=24)
    assert q.data_ptr() == out.data_ptr()
    whole[:, 1:, :DH] = 5.0
    assert bool((whole == 5.0).all())


@pytest.mark.gpu
def test_append_leaves_padding_rows(dev):
    """Rows behind the last request: their queries keep what ``out`` held, nothing is stored."""
    print("[gpu] paged append padding", flush=True)
    s = Step(dev, [3, 0, 4], [20, 4, 4], hkv=2, seed=5, pad=30, data=False)
    out = torch.full((s.T, 4, DH), 7.0, dtype=BF, device=dev)
    _check_append(s, 4, out=out, norms=True)
    assert bool((out[s.rows:] == 7.0).all()) and not bool((out[:s.rows] == 7.0).all())


@pytest.mark.gpu
def test_append_skips_what_has_no_place(dev):
    """Tokens whose page id is outside the pool, or past the table, are not stored; their queries
    are rotated all the same. A request whose length is smaller than its rows has its first rows
    left out."""
    print("[gpu] paged append bad pages", flush=True)
    s = Step(dev, [20, 4, 3], [40, 4, 3], hkv=2, seed=6, data=False)
    table = s.table.clone()
    table[0, 1], table[1, 0] = -5, 2**30  # tokens 16 .. 31 of request 0, all of request 1
    lens = torch.tensor([40, 4, 2], dtype=torch.int32, device=dev)
    batch = PagedBatch(table.to(dev), s.batch.q_start, lens, rows=s.rows, max_new=20, max_len=40)
    qkv = s.rand(s.T, 8 * DH)
    q = paged_append(qkv, s.k, s.v, batch, heads=4, theta=1e4,
                     out=torch.zeros(s.T, 4, DH, dtype=BF, device=dev))
    written = ~torch.isnan(s.v[:, 0, :, 0])
    assert int(written.sum()) == (40 - 32) + 0 + 2
    assert int((~torch.isnan(s.k)).sum()) == 10 * 2 * DH
    assert bool((q[24] == 0).all()) and bool((q[:24].abs().sum((1, 2)) > 0).all())
    cut = PagedBatch(s.table[:, :1].contiguous().to(dev), s.batch.q_start, s.batch.lens,
                     rows=s.rows, max_new=20, max_len=16)
    s.k.fill_(float("nan")), s.v.fill_(float("nan"))
    paged_append(qkv, s.k, s.v, cut, heads=4, theta=1e4)
    assert int((~torch.isnan(s.v[:, 0, :, 0])).sum()) == 0 + 4 + 3


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def _attend_reference(s, q, scale=None):
    """(rows, heads, 128) float64 and the error bound of the result before its own rounding."""
    hq = q.shape[1]
    hpg, scale = hq // s.hkv, scale or 1 / math.sqrt(DH)
    out = torch.zeros(s.rows, hq, DH, dtype=torch.float64, device=s.dev)
    tol = torch.zeros_like(out)
    # a score: 128 products summed in fp32, of size at most a; then the softmax's weight to bf16
    # (its half step is the larger one; fp16's is smaller) and the rest of the softmax in fp32
    half = torch.finfo(s.dtype).eps / 2
    for b, (m, n) in enumerate(zip(s.new, s.lens)):
        if m == 0:
            continue
        r = slice(s.starts[b], s.starts[b] + m)
        dead = (torch.arange(n, device=s.dev)[None, :]
                > torch.arange(n - m, n, device=s.dev)[:, None])
        for h in range(hq):
            k, v = s.tokens(s.k, b, h // hpg), s.tokens(s.v, b, h // hpg)
            z = (q[r, h].double() @ k.T) * scale
            p = torch.softmax(z.masked_fill(dead, -math.inf), -1)
            a = ((q[r, h].double().abs() @ k.abs().T) * scale).masked_fill(dead, 0).amax(-1)
            out[r, h] = p @ v
            rel = half + 2 * 130 * 2.0**-24 * a[:, None] + 2.0**-18
            tol[r, h] = rel * (p @ v.abs())
    return out, tol


def _check_attend(s, hq, *, scale=None, qscale=1.0, q=None):
    if q is None:
        q = s.rand(s.T, hq, DH, scale=qscale)
    want, tol = _attend_reference(s, q, scale)
    got = paged_attention(q, s.k, s.v, s.batch, scale=scale, out_dtype=torch.float32)
    err = (got[:s.rows].double() - want).abs()
    print(f"[gpu]   err/tol {float((err / (tol + 1e-30)).max()):.3f}", flush=True)
    assert bool((err <= tol + 1e-30).all())
    got16 = paged_attention(q, s.k, s.v, s.batch, scale=scale)
    assert got16.dtype == s.dtype and torch.equal(got16[:s.rows], got[:s.rows].to(s.dtype))
    return got


ATTEND = {
    # name: (new tokens, lengths, query heads, KV heads, page, dtype, layout)
    "one_key": ([1], [1], 4, 2, 16, BF, "plain"),
    "lens_around_tiles": ([1] * 8, [15, 16, 17, 63, 64, 65, 127, 129], 8, 2, 16, BF, "plain"),
    "step_fp16": ([1] * 5, [1, 300, 77, 1023, 512], 32, 8, 32, FP, "plain"),
    "step_long": ([1, 1], [8195, 5000], 32, 8, 64, BF, "plain"),
    "one_long": ([1], [20011], 8, 8, 128, FP, "plain"),
    "hpg16": ([1, 1, 1], [700, 31, 1500], 32, 2, 16, BF, "plain"),
    "hpg7_drafts": ([5, 2, 7], [500, 90, 7], 14, 2, 16, FP, "plain"),
    "drafts_long": ([4, 3], [6000, 4097], 8, 2, 32, BF, "plain"),
    "hpg3_prompt": ([100, 33], [100, 33], 6, 2, 16, BF, "plain"),
    "prompt": ([257, 64], [257, 64], 8, 2, 64, FP, "plain"),
    "prompt_odd": ([333, 1, 190], [333, 1, 190], 4, 4, 128, BF, "plain"),
    "chunk": ([130, 61], [1500, 61], 8, 2, 16, BF, "plain"),
    "chunk_long": ([40], [9001], 8, 2, 32, FP, "plain"),
    "mixed": ([1, 1, 150, 1, 0, 3, 1], [400, 17, 700, 1, 9, 2000, 64], 8, 2, 32, BF, "plain"),
    "heads_first": ([1, 70], [130, 95], 8, 2, 32, FP, "heads_first"),
    "pages_apart": ([1, 70, 2], [130, 95, 600], 16, 1, 16, BF, "apart"),
    "none_at_all": ([0, 2, 0], [5, 2, 0], 4, 1, 16, BF, "plain"),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(ATTEND))
def test_attention(dev, name):
    new, lens, hq, hkv, ps, dt, layout = ATTEND[name]
    print(f"[gpu] paged attention {name}", flush=True)
    _check_attend(Step(dev, new, lens, hkv=hkv, ps=ps, dtype=dt, layout=layout, seed=11), hq)


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1, 1], [700, 90]), ([80, 5], [300, 200])])
def test_attention_peaked_and_scaled(dev, new, lens):
    """A near one-hot softmax (the running maximum rises late), and a scale of its own."""
    print(f"[gpu] paged attention peaked {new}", flush=True)
    _check_attend(Step(dev, new, lens, hkv=2, seed=12), 8, qscale=8.0)
    _check_attend(Step(dev, new, lens, hkv=2, seed=13, dtype=FP), 8, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1] * 3, [700, 90, 33]), ([80, 5], [300, 200])])
def test_attention_leaves_padding_rows(dev, new, lens):
    print(f"[gpu] paged attention padding {new}", flush=True)
    s = Step(dev, new, lens, hkv=2, seed=14, pad=9)
    q = s.rand(s.T, 8, DH)
    want, tol = _attend_reference(s, q)
    whole = torch.full((s.T, 9, 2 * DH), 3.0, dtype=torch.float32, device=dev)
    out = whole[:, :8, :DH]
    got = paged_attention(q, s.k, s.v, s.batch, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert bool(((out[:s.rows].double() - want).abs() <= tol + 1e-30).all())
    out[:s.rows] = 3.0
    assert bool((whole == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 3, 60])
def test_attention_masks_pages_that_are_not_there(dev, new):
    """A page id outside the pool: its keys are masked. No page at all, or a length of zero: 0."""
    print(f"[gpu] paged attention bad pages {new}", flush=True)
    s = Step(dev, [new] * 4, [150, 150, 150, 60], hkv=2, seed=15)
    q = s.rand(s.T, 4, DH)
    want, _ = _attend_reference(s, q)
    s.table[1, 2], s.table[1, 5] = -1, 10**6      # tokens 32 .. 47 and 80 .. 95 of request 1
    s.table[2] = -1                               # all of request 2
    lens = torch.tensor([150, 150, 150, 0], dtype=torch.int32, device=dev)
    batch = PagedBatch(s.table.to(dev), s.batch.q_start, lens, rows=s.rows, max_new=new,
                       max_len=150, min_new=new)
    got = paged_attention(q, s.k, s.v, batch, out_dtype=torch.float32)
    pos = torch.arange(150 - new, 150, device=dev)[:, None]
    key = torch.arange(150, device=dev)[None]
    dead = (key > pos) | ((key // 16) == 2) | ((key // 16) == 5)
    good = [int(i) if 0 <= int(i) < s.k.shape[0] else 0 for i in s.table[1, :10]]
    for h in range(4):
        k = s.k[good, h // 2].reshape(-1, DH)[:150].double().nan_to_num()
        v = s.v[good, h // 2].reshape(-1, DH)[:150].double().nan_to_num()
        z = (q[new:2 * new, h].double() @ k.T / math.sqrt(DH)).masked_fill(dead, -math.inf)
        p = torch.softmax(z, -1)
        tol = 2.0**-7 * (p @ v.abs()) + 1e-30
        assert bool(((got[new:2 * new, h].double() - p @ v).abs() <= tol).all())
        err = (got[:new, h].double() - want[:new, h]).abs()
        assert bool((err <= 2.0**-7 * 4).all())
    assert bool((got[2 * new:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new,n,hkv", [(4, 300, 2), (60, 60, 2), (60, 3000, 2), (700, 700, 8)])
def test_attention_keeps_later_tokens_out(dev, new, n, hkv, value):
    """An infinity or NaN in a new token's key and value: the tokens before it, that do not attend
    it, have the result they have without it; the ones from it on have it in theirs."""
    print(f"[gpu] paged attention later {value} {new}", flush=True)
    s = Step(dev, [new, 1], [n, 40], hkv=hkv, seed=17)
    q = s.rand(s.T, 4 * hkv, DH)
    clean = paged_attention(q, s.k, s.v, s.batch, out_dtype=torch.float32)
    _, tol = _attend_reference(s, q)
    bad = n - new + new // 2  # the position of the token
    page, slot = int(s.table[0, bad // 16]), bad % 16
    s.v[page, :, slot, ::3] = value
    got = paged_attention(q, s.k, s.v, s.batch, out_dtype=torch.float32)
    before, after = slice(0, new // 2), slice(new // 2, new)
    assert bool(((got[before] - clean[before]).abs() <= 2 * tol[before]).all())
    assert torch.equal(got[new:], clean[new:])
    assert not bool(torch.isfinite(got[after][..., ::3]).any())
    # the dims beside it are what they were (a sum of their own)
    assert bool(((got[after] - clean[after]).abs() <= 2 * tol[after])[..., 1::3].all())
    s.k[page, :, slot] = value
    got = paged_attention(q, s.k, s.v, s.batch, out_dtype=torch.float32)
    assert bool(((got[before] - clean[before]).abs() <= 2 * tol[before]).all())
    assert torch.equal(got[new:], clean[new:])


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1, 1], [900, 450]), ([90, 2], [350, 200])])
def test_attention_same_result_every_time(dev, new, lens):
    print(f"[gpu] paged attention repeat {new}", flush=True)
    s = Step(dev, new, lens, hkv=2, seed=16)
    q = s.rand(s.T, 8, DH)
    first = paged_attention(q, s.k, s.v, s.batch)
    for _ in range(3):
        assert torch.equal(paged_attention(q, s.k, s.v, s.batch), first)
    strided = torch.empty(s.T, 8, 2, DH, dtype=BF, device=dev)[:, :, 1]
    strided.copy_(q)
    assert torch.equal(paged_attention(strided, s.k, s.v, s.batch), first)


def _random_step(i):
    g = torch.Generator().manual_seed(500 + i)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    hkv = [1, 2, 3, 8][r(0, 3)]
    hq = hkv * [1, 2, 4, 5, 8, 16][r(0, 5)]
    n = r(1, 6)
    kind = r(0, 3)
    new = [[1, r(1, 6), r(1, 200), [0, 1, r(2, 90)][r(0, 2)]][kind] for _ in range(n)]
    if not any(new):
        new[0] = 1
    lens = [m + (0 if r(0, 2) == 0 else int(math.exp(float(torch.rand(1, generator=g)) * 8)))
            for m in new]
    return new, lens, hq, hkv, [16, 32, 64, 128, 256][r(0, 4)], [BF, FP][r(0, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(16))
def test_random_steps(dev, i):
    """Append, then attention, of a random step."""
    new, lens, hq, hkv, ps, dt = _random_step(i)
    print(f"[gpu] random step {i}: {new} {lens} {hq}/{hkv} page {ps} {dt}", flush=True)
    s = Step(dev, new, lens, hkv=hkv, ps=ps, dtype=dt, seed=600 + i)
    q = _check_append(s, hq, norms=i % 2 == 0)
    _check_attend(s, hq, q=q)


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_chunks_give_what_a_whole_prompt_gives(dev):
    """Three requests through a cache: prompts in chunks of different sizes beside single tokens,
    one request ended and its pages reused, one cut back; every output against attention over the
    request's tokens kept aside."""
    print("[gpu] paged chunks", flush=True)
    hq, hkv, theta = 8, 2, 10000.0
    cache = PagedKVCache(1, 24, hkv, page_size=16, device=dev)
    cache.k[0].fill_(float("nan")), cache.v[0].fill_(float("nan"))
    g = torch.Generator().manual_seed(77)
    rand = lambda n: torch.randn(n, (hq + 2 * hkv) * DH, generator=g).to(BF).to(dev)  # noqa: E731
    kept: dict = {}
    a, b, c = cache.add(), cache.add(), cache.add()

    def step(parts):
        qkv = rand(sum(n for _, n in parts))
        batch = cache.batch(parts)
        q = paged_append(qkv, cache.k[0], cache.v[0], batch, heads=hq, theta=theta)
        o = paged_attention(q, cache.k[0], cache.v[0], batch, out_dtype=torch.float32)
        at = 0
        for r, n in parts:
            kept[r] = torch.cat([kept[r], qkv[at:at + n]]) if r in kept else qkv[at:at + n]
            total = kept[r].shape[0]
            assert total == cache.length(r)
            x = kept[r].double().view(total, hq + 2 * hkv, DH)
            pos = torch.arange(total, dtype=torch.float64, device=dev)
            y = _turn(x[:, :hq + hkv], pos, _freq(dev, theta)).to(BF).double()
            for h in range(hq):
                z = y[total - n:, h] @ y[:, hq + h // 4].T / math.sqrt(DH)
                z.masked_fill_(torch.arange(total, device=dev)[None]
                               > torch.arange(total - n, total, device=dev)[:, None], -math.inf)
                v = x[:, hq + hkv + h // 4]
                p = torch.softmax(z, -1)
                # a key or query may round to the other neighbour: one step of one of 128 products
                # moves a score by at most 2^-7 |q||k| / sqrt(128); 2^-6 covers it and the weights
                assert bool(((o[at:at + n, h].double() - p @ v).abs()
                             <= 2.0**-6 * (p @ v.abs()) + 2.0**-7).all()), (r, total, h)
            at += n

    step([(a, 70), (b, 5)])
    step([(b, 40), (a, 1)])
    step([(a, 1), (c, 100), (b, 1)])
    cache.truncate(c, 90)
    kept[c] = kept[c][:90]
    step([(a, 1), (b, 0), (c, 3)])
    cache.free(a)
    d = cache.add()
    step([(d, 130), (c, 1), (b, 2)])
    step([(d, 1), (c, 1), (b, 1)])


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1] * 4, [700, 90, 33, 260]), ([60, 1, 9], [300, 200, 100])])
def test_captured_step(dev, new, lens):
    """A captured append and attention, replayed with other inputs, lengths and pages in the same
    buffers, with eager work between the replays; two graphs replayed at once on two streams."""
    print(f"[gpu] paged graph {new}", flush=True)
    side = torch.cuda.Stream()
    s = [Step(dev, new, lens, hkv=2, seed=21 + i) for i in range(2)]
    qkv = [t.rand(t.T, 12 * DH) for t in s]
    one = lambda i: paged_attention(  # noqa: E731
        paged_append(qkv[i], s[i].k, s[i].v, s[i].batch, heads=8, theta=1e4), s[i].k, s[i].v,
        s[i].batch)
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for i in range(2):
            one(i)
        torch.cuda.synchronize()
        for i in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                outs.append(one(i))
            graphs.append(gr)
    torch.cuda.synchronize()
    other = Step(dev, [1], [3000], hkv=2, seed=29)
    oq = other.rand(1, 8, DH)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        for i in range(2):
            qkv[i].copy_(s[i].rand(s[i].T, 12 * DH))
            if rep == 2:  # shorter, and two pages changed places
                t = s[i]
                t.lens = [max(m, n - 20) for m, n in zip(t.new, t.lens)]
                t.batch.lens.copy_(torch.tensor(t.lens, dtype=torch.int32))
                t.table[0, [0, 1]] = t.table[0, [1, 0]]
                t.batch.page_table.copy_(t.table)
        paged_attention(oq, other.k, other.v, other.batch)
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for i in range(2):
            got, k, v = outs[i].clone(), s[i].k.clone(), s[i].v.clone()
            assert torch.equal(one(i), got), (rep, i)
            assert torch.equal(s[i].k.view(torch.int16), k.view(torch.int16))
            assert torch.equal(s[i].v.view(torch.int16), v.view(torch.int16))


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    print("[gpu] paged two streams", flush=True)
    s = [Step(dev, [1, 2], [1500, 1100 + 300 * i], hkv=2, seed=31 + i) for i in range(2)]
    q = [t.rand(t.T, 8, DH) for t in s]
    want = [paged_attention(q[i], s[i].k, s[i].v, s[i].batch) for i in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged_attention(q[i], s[i].k, s[i].v, s[i].batch))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


@pytest.mark.gpu
def test_pool_past_32_bits(dev):
    """Pages whose elements lie past 2^32 bytes of the pool's start."""
    print("[gpu] paged large pool", flush=True)
    ps, hkv, pages = 256, 2, 40000  # 5.2 GB each for keys and values
    k = torch.empty(pages, hkv, ps, DH, dtype=BF, device=dev)
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(41)
    for new, n in ((1, 700), (70, 700)):
        ids = torch.tensor([[pages - 1, 3, pages - 900]], dtype=torch.int32)
        for i in ids[0].tolist():
            k[i] = torch.randn(hkv, ps, DH, generator=g).to(BF)
            v[i] = torch.randn(hkv, ps, DH, generator=g).to(BF)
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        batch = PagedBatch(ids.to(dev), i32(0, new), i32(n), rows=new, max_new=new, max_len=n,
                           min_new=new)
        small = Step(dev, [new], [n], hkv=hkv, ps=ps, seed=42)
        qkv = small.rand(new, 8 * DH)
        order = small.table[0, :3].long().to(dev)
        small.k[order], small.v[order] = k[ids[0].long().to(dev)], v[ids[0].long().to(dev)]
        qa = paged_append(qkv, k, v, batch, heads=4, theta=1e4)
        qb = paged_append(qkv, small.k, small.v, small.batch, heads=4, theta=1e4)
        assert torch.equal(qa, qb) and torch.equal(k[ids[0].long().to(dev)], small.k[order])
        assert torch.equal(v[ids[0].long().to(dev)], small.v[order])
        assert torch.equal(paged_attention(qa, k, v, batch),
                           paged_attention(qb, small.k, small.v, small.batch))


MANY = {
    # more requests than one wave holds the lengths of: a workgroup each, single or with prompts beside
    "single": ([1, 1, 0] * 100, [40, 300, 7] * 100, 8, 2, 16),
    "mixed": ([1, 40, 0, 2] * 70, [90, 41, 5, 700] * 70, 8, 2, 32),
    "prompts": ([17, 40] * 140, [17, 60] * 140, 4, 2, 16),
    # more (request, KV head) units than counters
    "units": ([1] * 256, [20, 70] * 128, 65, 65, 16),
    "large_pages": ([1, 90, 1], [3000, 1500, 1025], 8, 2, 1024),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(MANY))
def test_attention_many_requests_and_large_pages(dev, name):
    new, lens, hq, hkv, ps = MANY[name]
    print(f"[gpu] paged attention many {name}", flush=True)
    s = Step(dev, new, lens, hkv=hkv, ps=ps, seed=51)
    q = s.rand(s.T, hq, DH)
    got = paged_attention(q, s.k, s.v, s.batch, out_dtype=torch.float32)
    want, tol = _attend_reference(_First(s, 6), q)
    n = want.shape[0]
    assert bool(((got[:n].double() - want).abs() <= tol + 1e-30).all())
    # the requests behind: the same keys alone give the same within both bounds
    for b in {len(new) - 1, len(new) // 2}:
        one = PagedBatch(s.batch.page_table[b:b + 1], torch.tensor([0, new[b]], dtype=torch.int32,
                                                                   device=dev),
                         s.batch.lens[b:b + 1], rows=new[b], max_new=new[b], max_len=lens[b],
                         min_new=new[b])
        r = slice(s.starts[b], s.starts[b + 1])
        alone = paged_attention(q[r], s.k, s.v, one, out_dtype=torch.float32)
        size = max(float(s.tokens(s.v, b, g).abs().max()) for g in range(hkv)) if new[b] else 0.0
        assert bool(((got[r] - alone).abs() <= 2 * (2.0**-8 + 2.0**-12) * size).all())


class _First:
    """The first requests of a step, for the reference."""

    def __init__(self, s, n):
        self.s, self.new, self.lens = s, s.new[:n], s.lens[:n]
        self.rows, self.starts = s.starts[len(self.new)], s.starts

    def __getattr__(self, name):
        return getattr(self.s, name)


@pytest.mark.gpu
def test_steps_of_nothing(dev):
    print("[gpu] paged empty steps", flush=True)
    cache = PagedKVCache(1, 4, 2, page_size=16, device=dev)
    a = cache.add()
    for step in ([], [(a, 0)]):
        batch = cache.batch(step)
        qkv = torch.randn(3, 8 * DH, device=dev).to(BF)  # rows of no request
        out = torch.full((3, 4, DH), 2.0, dtype=BF, device=dev)
        q = paged_append(qkv, cache.k[0], cache.v[0], batch, heads=4, theta=1e4, out=out)
        o = paged_attention(q, cache.k[0], cache.v[0], batch, out=out)
        assert bool((o == 2.0).all())
        none = paged_append(qkv[:0], cache.k[0], cache.v[0], batch, heads=4, theta=1e4)
        assert paged_attention(none, cache.k[0], cache.v[0], batch).shape == (0, 4, DH)


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1, 1], [700, 90]), ([3, 2], [300, 900]),
                                      ([80, 5, 1], [300, 200, 50]), ([40], [5000])])
def test_in_place(dev, new, lens):
    """The queries rotated in the projection's own columns, the output written over the queries."""
    print(f"[gpu] paged in place {new}", flush=True)
    s = Step(dev, new, lens, hkv=2, seed=52)
    qkv = s.rand(s.T, 12 * DH)
    q = paged_append(qkv, s.k, s.v, s.batch, heads=8, theta=1e4)
    k, v = s.k.clone(), s.v.clone()
    o = paged_attention(q, s.k, s.v, s.batch)
    mine = qkv[:, :8 * DH].view(s.T, 8, DH)
    assert paged_append(qkv, s.k, s.v, s.batch, heads=8, theta=1e4, out=mine) is mine
    assert torch.equal(mine, q)
    assert torch.equal(s.k.view(torch.int16), k.view(torch.int16))
    assert torch.equal(s.v.view(torch.int16), v.view(torch.int16))
    assert paged_attention(mine, s.k, s.v, s.batch, out=mine) is mine
    assert torch.equal(mine, o)


@pytest.mark.gpu
def test_strides_of_single_rows_and_shared_queries(dev):
    print("[gpu] paged odd strides", flush=True)
    s = Step(dev, [1], [77], hkv=2, seed=53)
    row = s.rand(1, 12 * DH)
    odd = torch.empty(12 * DH, 1, dtype=BF, device=dev).t()  # a row stride of 1
    odd.copy_(row)
    q = paged_append(row, s.k, s.v, s.batch, heads=8, theta=1e4)
    out = torch.empty_strided((1, 8, DH), (3, DH, 1), dtype=BF, device=dev)
    assert torch.equal(paged_append(odd, s.k, s.v, s.batch, heads=8, theta=1e4, out=out), q)
    want = paged_attention(q, s.k, s.v, s.batch)
    got = torch.empty_strided((1, 8, DH), (3, DH, 1), dtype=torch.float32, device=dev)
    paged_attention(out, s.k, s.v, s.batch, out=got)
    assert torch.equal(got.to(BF), want)
    for new, lens in (([2, 1], [90, 33]), ([70, 1], [90, 33])):
        s = Step(dev, new, lens, hkv=2, seed=54)
        one = s.rand(s.T, 1, DH).expand(s.T, 8, DH)
        want = paged_attention(one.contiguous(), s.k, s.v, s.batch)
        assert torch.equal(paged_attention(one, s.k, s.v, s.batch), want)
        # heads first, in fp32, at an odd offset: rows that 16 bytes do not divide
        wide = torch.full((8, s.T, DH + 1), 5.0, dtype=torch.float32, device=dev)
        out = wide[..., 1:].transpose(0, 1)
        paged_attention(one, s.k, s.v, s.batch, out=out)
        assert torch.equal(out.to(BF), want) and bool((wide[..., 0] == 5.0).all())
        # queries whose rows are not aligned
        skew = torch.empty(s.T * 8 * DH + 3, dtype=BF, device=dev)[3:].view(s.T, 8, DH)
        skew.copy_(one)
        assert torch.equal(paged_attention(skew, s.k, s.v, s.batch), want)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 3, 60])
def test_lengths_past_the_table_and_shared_pages(dev, new):
    """A length the table has no room for ends with it, and a page that two requests hold (or one
    of them twice) is read by both."""
    print(f"[gpu] paged shared pages {new}", flush=True)
    s = Step(dev, [new, new], [128, 96], hkv=2, seed=55)
    q = s.rand(s.T, 4, DH)
    s.table[1, :6] = s.table[0, :6]
    s.table[1, 3] = s.table[1, 2]
    table = s.table[:, :8].contiguous().to(dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    batch = PagedBatch(table, s.batch.q_start, i32(128 + 40, 96), rows=s.rows, max_new=new,
                       max_len=128, min_new=new)
    got = paged_attention(q, s.k, s.v, batch, out_dtype=torch.float32)
    for b, n, end in ((0, 128, 168), (1, 96, 96)):
        ids = s.table[b, :n // 16].long().to(dev)
        pos = torch.arange(end - new, end, device=dev)[:, None]
        dead = torch.arange(n, device=dev)[None] > pos
        r = slice(b * new, (b + 1) * new)
        for h in range(4):
            k, v = (x[ids, h // 2].reshape(-1, DH).double() for x in (s.k, s.v))
            z = (q[r, h].double() @ k.T / math.sqrt(DH)).masked_fill(dead, -math.inf)
            p = torch.softmax(z, -1)
            assert bool(((got[r, h].double() - p @ v).abs() <= 2.0**-7 * (p @ v.abs())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1, 1], [700, 90]), ([3], [40]), ([80, 1], [300, 50]),
                                      ([40], [5000])])
def test_attention_scores_of_any_size(dev, new, lens):
    """Scores far below zero (all of them), a NaN score (its row is NaN), an infinite one."""
    print(f"[gpu] paged attention scores {new}", flush=True)
    s = Step(dev, new, lens, hkv=2, seed=56)
    q = torch.zeros(s.T, 8, DH, dtype=BF, device=dev)
    q[..., 0] = 2.0**60
    ids = [int(s.table[b, t]) for b, n in enumerate(lens) for t in range(-(-n // 16))]
    s.k[ids] = 0.0
    s.k[ids, :, :, 0] = -(2.0**62)
    first = int(s.table[0, 0])
    s.k[first, :, 0, 0] = -(2.0**61)  # the largest of request 0: its first key
    got = paged_attention(q, s.k, s.v, s.batch)
    want = s.v[first, :, 0].repeat_interleave(4, 0)
    assert torch.equal(got[:new[0]], want.expand(new[0], 8, DH))
    # all alike: the mean of the values
    if len(new) > 1:
        r, n = s.starts[1], lens[1]
        mean = torch.stack([s.tokens(s.v, 1, h // 4)[:n - new[1] + 1].mean(0) for h in range(8)])
        size = torch.stack([s.tokens(s.v, 1, h // 4)[:n - new[1] + 1].abs().mean(0)
                            for h in range(8)])
        assert bool(((got[r].double() - mean).abs() <= 2.0**-7 * size).all())
    q = s.rand(s.T, 8, DH)
    base = paged_attention(q, s.k, s.v, s.batch)
    for value in (math.nan, math.inf):
        bad = q.clone()
        bad[0, 3, 5] = value
        got = paged_attention(bad, s.k, s.v, s.batch)
        if value != value:
            assert bool(torch.isnan(got[0, 3]).all())
        got[0, 3] = base[0, 3]
        assert torch.equal(got, base)
    k = s.k.clone()
    k[first, 0, 0] = math.nan  # a key that every row of request 0 attends
    got = paged_attention(q, k, s.v, s.batch)
    assert bool(torch.isnan(got[:new[0], :4]).all())
    got[:new[0], :4] = base[:new[0], :4]
    assert torch.equal(got, base)


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [dict(min_new=5), dict(max_len=20000), dict(max_new=80)])
def test_attention_loose_bounds(dev, odd):
    """Bounds choose the launch alone: any that hold give the same within the roundings, and a least
    number of new tokens that does not hold costs no row."""
    print(f"[gpu] paged attention bounds {odd}", flush=True)
    s = Step(dev, [1, 40, 0, 4], [700, 90, 12, 3000], hkv=2, seed=57)
    q = s.rand(s.T, 8, DH)
    want, tol = _attend_reference(s, q)
    table = torch.cat([s.table, torch.full((4, 1300), -1, dtype=torch.int32)], 1).to(dev)
    rows = max(s.rows, odd.get("max_new", 0))
    q2 = torch.cat([q, s.rand(rows - s.rows, 8, DH)])
    batch = PagedBatch(table, s.batch.q_start, s.batch.lens,
                       **(dict(rows=rows, max_new=40, max_len=3000, min_new=1) | odd))
    got = paged_attention(q2, s.k, s.v, batch, out_dtype=torch.float32)[:s.rows]
    assert bool(((got.double() - want).abs() <= tol + 1e-30).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1, 1], [700, 90]), ([3], [400]), ([80, 1], [300, 50]),
                                      ([40], [5000]), ([257], [257])])
@pytest.mark.parametrize("size", [2.0**13, 2.0**30, 2.0**50])
def test_attention_scores_far_apart(dev, new, lens, size):
    """Scores so large that the softmax is one key's: the output is that key's value exactly, for each
    row whose two largest scores differ by more than fp32 sums can be off by."""
    print(f"[gpu] paged attention far apart {new} {size}", flush=True)
    s = Step(dev, new, lens, hkv=2, seed=58)
    ids = sorted({int(i) for b, n in enumerate(lens) for i in s.table[b, :-(-n // 16)]})
    s.k[ids] = s.k[ids] * size
    q = s.rand(s.T, 8, DH, scale=size)
    got = paged_attention(q, s.k, s.v, s.batch)
    checked = 0
    for b, (m, n) in enumerate(zip(new, lens)):
        pos = torch.arange(n - m, n, device=dev)[:, None]
        dead = torch.arange(n, device=dev)[None] > pos
        r = slice(s.starts[b], s.starts[b] + m)
        for h in range(8):
            k, v = s.tokens(s.k, b, h // 4), s.tokens(s.v, b, h // 4)
            z = (q[r, h].double() @ k.T / math.sqrt(DH)).masked_fill(dead, -math.inf)
            a = (q[r, h].double().abs() @ k.T.abs() / math.sqrt(DH)).masked_fill(dead, 0).amax(-1)
            top, at = torch.cat([z, z[:, :1] * 0 - math.inf], 1).topk(2)
            # off by 130 roundings each, and 40 more halvings than bf16 can show
            sure = top[:, 0] - top[:, 1] > 2 * 130 * 2.0**-24 * a + 40
            assert torch.equal(got[r, h][sure], v.to(BF)[at[:, 0]][sure]), (b, h)
            checked += int(sure.sum())
    assert checked > 0.9 * s.rows * 8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_same_with_and_without_the_tensor_module(dev, dtype, monkeypatch):
    print(f"[gpu] paged without the tensor module {dtype}", flush=True)
    s = [Step(dev, new, lens, hkv=2, seed=59, dtype=dtype, pad=2)
         for new, lens in (([1], [90]), ([1, 1], [700, 90]), ([40, 3], [60, 9]), ([0, 2], [4, 7]))]
    inputs = [(t.rand(t.T, 12 * DH), 1 + t.rand(DH, scale=0.2)) for t in s]

    def run():
        out = []
        for t, (qkv, w) in zip(s, inputs):
            q = paged_append(qkv, t.k, t.v, t.batch, heads=8, theta=1e4)
            q2 = paged_append(qkv, t.k, t.v, t.batch, heads=8, inv_freq=[0.5] * 64, q_norm=w, k_norm=w,
                              eps=1e-5)
            o = paged_attention(q2, t.k, t.v, t.batch)
            out += [x[:t.rows] for x in (q, q2, o, paged_attention(q, t.k, t.v, t.batch, scale=0.2))]
        return [x.clone() for x in out] + [t.k.view(torch.int16).clone() for t in s]

    fast = run()
    monkeypatch.setattr(_lib, "_tensor_calls", None)
    for a, b in zip(run(), fast):
        assert a.dtype == b.dtype and torch.equal(a, b)
    with torch.cuda.stream(torch.cuda.Stream()):
        monkeypatch.setattr(_lib, "_tensor_calls", False)
        torch.cuda.synchronize()
        for a, b in zip(run(), fast):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [14, 16, 18])
@pytest.mark.parametrize("new,lens", [([1, 1], [4000, 9001]), ([3], [4000]), ([40], [4000]),
                                      ([300, 1], [4000, 700]), ([70], [70])])
def test_fp16_weights_far_below_the_largest(dev, new, lens, gap):
    """A first key ``gap`` nats above all others, whose value is 0: the output is the others', whose
    weights are 2^-20 to 2^-26 of the largest. An fp16 weight's step is 2^-24 below 2^-14, so a row's
    largest weight is kept at 2^12 or more: a weight is off by at most 2^-25 of 2^12, or by its own half
    step, which ``_attend_reference`` counts."""
    print(f"[gpu] paged attention far below {new} {gap}", flush=True)
    s = Step(dev, new, lens, hkv=2, seed=61, dtype=FP)
    q = s.rand(s.T, 8, DH, scale=0.3)
    q[..., 0] = 8.0
    for b, n in enumerate(lens):
        ids = s.table[b, :-(-n // 16)].tolist()
        s.k[ids, :, :, 0] = torch.where(s.k[ids, :, :, 0].isnan(), s.k[ids, :, :, 0], 0.0)
        s.v[ids] += 0.5
        s.k[ids[0], :, 0] = 0.0
        s.k[ids[0], :, 0, 0] = gap * math.sqrt(DH) / 8.0
        s.v[ids[0], :, 0] = 0.0
    want, tol = _attend_reference(s, q)
    for b, (m, n) in enumerate(zip(new, lens)):  # the largest weight is at most 1
        for h in range(8):
            size = s.tokens(s.v, b, h // 4).abs().sum(0)
            tol[s.starts[b]:s.starts[b] + m, h] += 2.0**-37 * size
    got = paged_attention(q, s.k, s.v, s.batch, out_dtype=torch.float32)
    err = (got.double() - want).abs()
    print(f"[gpu]   err/tol {float((err / (tol + 1e-30)).max()):.3f}", flush=True)
    assert bool((err <= tol + 1e-30).all())
    assert torch.equal(paged_attention(q, s.k, s.v, s.batch), got.to(FP))


@pytest.mark.gpu
def test_threads_on_one_stream(dev):
    """Calls from several threads on one stream, of one launch and of two (key ranges and their join):
    each has its own result."""
    print("[gpu] paged threads", flush=True)
    s = [Step(dev, new, lens, hkv=2, seed=63 + i) for i, (new, lens) in enumerate(
        (([40], [3000]), ([64], [2500]), ([1, 1, 40], [900, 450, 2000]), ([1, 1], [2000, 700])))]
    q = [t.rand(t.T, 8, DH) for t in s]
    want = [paged_attention(q[i], t.k, t.v, t.batch) for i, t in enumerate(s)]
    torch.cuda.synchronize()
    got = [[] for _ in s]

    def run(i):
        for _ in range(60):
            got[i].append(paged_attention(q[i], s[i].k, s[i].v, s[i].batch))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(s))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(len(s)):
        assert len(got[i]) == 60 and all(torch.equal(o, want[i]) for o in got[i]), i


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens,bounds", [
    ([0] * 30 + [64] + [0] * 9, [40] * 30 + [3000] + [700] * 9, {}),
    ([0] * 30 + [64, 1] + [0] * 9, [40] * 30 + [3000, 90] + [700] * 9, {}),
    # a least number of new tokens that does not hold: more row tiles than it allows for
    ([1] * 20 + [64], [500, 17] * 10 + [3000], dict(min_new=64)),
])
def test_attention_beside_requests_of_no_new_token(dev, new, lens, bounds):
    print(f"[gpu] paged attention idle requests {len(new)} {bounds}", flush=True)
    s = Step(dev, new, lens, hkv=2, seed=67)
    q = s.rand(s.T, 8, DH)
    want, tol = _attend_reference(s, q)
    batch = PagedBatch(s.batch.page_table, s.batch.q_start, s.batch.lens, **(dict(
        rows=s.rows, max_new=64, max_len=3000, min_new=s.batch.min_new) | bounds))
    got = paged_attention(q, s.k, s.v, batch, out_dtype=torch.float32)
    assert bool(((got.double() - want).abs() <= tol + 1e-30).all())


@pytest.mark.gpu
def test_a_cache_stays_on_its_device(dev):
    """A cache made for "cuda" is on the device that was current then, and its batches go there whichever
    is current later."""
    print("[gpu] paged cache device", flush=True)
    cache = PagedKVCache(1, 4, 2, page_size=16, device="cuda")
    assert cache.device == cache.k[0].device and cache.device.index is not None
    a = cache.add()
    assert cache.batch([(a, 3)]).page_table.device == cache.device
