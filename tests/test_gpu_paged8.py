"""Pages of 8 bits on the GPU: the append to them, the attention over them and pages read back, against
the formulas in float64.

Pools start full of NaN codes and NaN scales and tables end in ids outside the pool, so what is read
without having been written shows; an append is checked by comparing whole pools, codes and scales.
Codes are whole numbers: values have to get the nearest one exactly, keys too but where the float64
value is within its own error of a border between two. The attention's tolerance is the 16-bit
one's (``_attend_reference``): codes times scales are numbers of the queries' type, so the pages'
values enter without a rounding."""
import math

import pytest
import torch

from dynakv_amd.kernels.paged import (PagedBatch, PagedKVCache, paged_append, paged_attention,
                                      paged_values)
from test_gpu_paged import (BF, DH, FP, Step, _append_reference, _append_tol, _attend_reference,
                            _freq, _turn)

CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu
BLOCK = 16
RANGE = {FP: (-15, 7), BF: (-110, 119)}
GRID = torch.tensor([i / 512.0 for i in range(8)]
                    + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1],
                    dtype=torch.float64)  # the values of the codes 0 .. 126
# the reference's own error in a key, relative to its pair's size: products and sums in 64 bits, and the
# angle, up to 2^17 times a frequency, that two 64-bit roundings put off by 2^-34 of a radian at most
SLACK = 2.0**-33


def nearest(y):
    """The codes' value nearest to y (float64), ties to the even code, at most 448."""
    grid = GRID.to(y.device)
    a = y.abs().clamp(max=448.0).contiguous()
    lo = torch.searchsorted(grid, a, right=True) - 1
    hi = (lo + 1).clamp(max=126)
    down, up = a - grid[lo], grid[hi] - a
    pick = (up < down) | ((up == down) & (hi % 2 == 0))
    return torch.where(pick, grid[hi], grid[lo]).copysign(y)


def two_to(e):
    """2^e in float64 by its bits (a library's power may be off by a step)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


class Step8(Step):
    """A step over 8-bit pages: the requests' earlier tokens are held as random values are, with
    block scales some powers of two apart; the new ones too where ``data``."""

    def __init__(self, dev, new, lens, *, spread=3, unit=0, layout="plain", data=True, **kw):
        self.layout = layout
        super().__init__(dev, new, lens, layout=layout, data=False, **kw)
        pages = self.k.shape[0]
        self.k_scale, self.v_scale = self.scales(pages), self.scales(pages)
        for b, n in enumerate(lens):
            if not data:
                n -= new[b]
            for t0 in range(0, n, BLOCK):
                m = min(BLOCK, n - t0)
                page, slot = int(self.table[b, t0 // self.ps]), t0 % self.ps
                for codes, scale in ((self.k, self.k_scale), (self.v, self.v_scale)):
                    e = torch.randint(-spread, spread + 1, (self.hkv,), generator=self.g) - 8 + unit
                    x = torch.randn(self.hkv, m, DH, generator=self.g) * 150.0
                    codes[page, :, slot:slot + m] = x.clamp(-448, 448).to(CODES).to(dev)
                    scale.view(torch.uint8)[page, :, slot // BLOCK] = (e + 127).to(
                        torch.uint8).to(dev)

    def pool(self, pages, layout):
        if layout == "heads_first":
            t = torch.full((self.hkv, pages, self.ps, DH), 0x7f, dtype=torch.uint8,
                           device=self.dev).transpose(0, 1)
        elif layout == "apart":
            t = torch.full((pages, self.hkv + 1, self.ps + 16, DH), 0xff, dtype=torch.uint8,
                           device=self.dev)[:, :self.hkv, :self.ps]
        else:
            t = torch.full((pages, self.hkv, self.ps, DH), 0x7f, dtype=torch.uint8,
                           device=self.dev)
        return t.view(CODES)

    def scales(self, pages):
        n = self.ps // BLOCK
        if self.layout == "heads_first":
            t = torch.full((self.hkv, pages, n), 255, dtype=torch.uint8,
                           device=self.dev).transpose(0, 1)
        elif self.layout == "apart":
            t = torch.full((pages, self.hkv + 2, n + 3), 255, dtype=torch.uint8,
                           device=self.dev)[:, 1:-1, 1:n + 1]
        else:
            t = torch.full((pages, self.hkv, n), 255, dtype=torch.uint8, device=self.dev)
        return t.view(SCALES)

    @property
    def both(self):
        return dict(k_scale=self.k_scale, v_scale=self.v_scale)

    def held(self, codes):
        """(pages, hkv, ps, 128) float64 values."""
        scale = self.k_scale if codes is self.k else self.v_scale
        e = scale.contiguous().view(torch.uint8).double() - 127
        two = torch.where(e == 128, math.nan, two_to(e))
        return codes.contiguous().double() * two.repeat_interleave(BLOCK, -1)[..., None]

    def tokens(self, pool, b, g):
        n = self.lens[b]
        ids = self.table[b, :-(-n // self.ps)].long().to(self.dev)
        if getattr(self, "_seen", None) is None:
            self._seen = {}
        key = (id(pool), b, g)
        if key not in self._seen:
            scale = (self.k_scale if pool is self.k else self.v_scale)[ids, g]
            e = scale.contiguous().view(torch.uint8).double() - 127
            two = torch.where(e == 128, math.nan, two_to(e))
            x = pool[ids, g].double() * two.repeat_interleave(BLOCK, -1)[..., None]
            self._seen[key] = x.reshape(-1, DH)[:n]
        return self._seen[key]

    def forget(self):
        self._seen = None


def u8(t):
    return t.contiguous().view(torch.uint8)


# ---------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------
def _check_block(s, name, codes0, scale0, page, g, i, first, y, slack):
    """One block after an append: old codes and exponent, the first new slot, new values (n, 128)."""
    codes = (s.k if name == "k" else s.v)[page, g, i * BLOCK:(i + 1) * BLOCK]
    e = int((s.k_scale if name == "k" else s.v_scale).view(torch.uint8)[page, g, i]) - 127
    low, high = RANGE[s.dtype]
    old_e = min(max(int(scale0[page, g, i]) - 127, low), high)
    fine = torch.isfinite(y)
    big = float(torch.where(fine, y, 0.0).abs().max())
    must = 2.0 ** e * 448 >= big * (1 - SLACK) or e == high
    least = low if first == 0 else max(low, old_e)
    could_be_less = e > least and 2.0 ** (e - 1) * 448 >= big * (1 + SLACK)
    assert low <= e <= high and e >= least and must and not could_be_less, (name, page, g, i, e, big)
    # earlier tokens: rounded again where the exponent rose
    was = codes0[page, g, i * BLOCK:i * BLOCK + first].view(CODES)
    if e > old_e:
        want = nearest(was.double() * 2.0 ** (old_e - e))
        want[was.double().isnan()] = math.nan
        got = codes[:first].double()
        assert bool(((got == want) | (got.isnan() & want.isnan())).all()), (name, page, g, i)
    else:
        assert torch.equal(u8(codes[:first]), u8(was))
    got = codes[first:first + y.shape[0]].double()
    x = y * 2.0 ** -e
    want = nearest(torch.where(fine, x, 0.0))
    assert torch.equal(got.isnan(), ~fine), (name, page, g, i)
    off = fine & (got != want)
    # another code only where the value is a border's neighbour within its own error
    border = (got + want) / 2
    near = (x - border).abs() <= slack * 2.0 ** -e
    assert bool((near | ~off).all()), (name, page, g, i, int((off & ~near).sum()))
    assert torch.equal(u8(codes[first + y.shape[0]:]),
                       codes0[page, g, i * BLOCK + first + y.shape[0]:(i + 1) * BLOCK])


def _check_append(s, heads, *, theta=500000.0, norms=False, qkv=None, out=None, weights=0.2):
    if qkv is None:
        qkv = s.rand(s.T, (heads + 2 * s.hkv) * DH)
    qn = kn = None
    if norms:
        qn, kn = 1 + s.rand(DH, scale=weights), 1 + s.rand(DH, scale=weights)
    before = {n: (u8(c).clone(), u8(e).clone()) for n, c, e in (("k", s.k, s.k_scale),
                                                               ("v", s.v, s.v_scale))}
    x0 = qkv.clone()
    q = paged_append(qkv, s.k, s.v, s.batch, heads=heads, theta=theta, q_norm=qn, k_norm=kn, out=out,
                     **s.both)
    wq, wk, wv, sq, sk = _append_reference(s, qkv, heads, _freq(s.dev, theta), qn, kn)
    assert torch.equal(qkv.view(torch.int16), x0.view(torch.int16))
    # (and fp16's numbers below 2^-14 are 2^-24 apart: half a step of those is 2^-25, whatever their size)
    tol = _append_tol(wq, sq, s.dtype) + (2.0**-25 if s.dtype == FP else 0.0)
    # (a rotation's result past the type's largest number has none to be rounded to)
    past = ~(wq.abs() <= torch.finfo(s.dtype).max)
    good = bool((((q[:s.rows].double() - wq).abs() <= tol) | past).all())
    assert good
    touched = {n: (torch.zeros_like(c, dtype=torch.bool), torch.zeros_like(e, dtype=torch.bool))
               for n, (c, e) in before.items()}
    at = 0
    for b, (m, n) in enumerate(zip(s.new, s.lens)):
        for t0 in range((n - m) // BLOCK * BLOCK, n, BLOCK):
            lo, hi = max(t0, n - m), min(t0 + BLOCK, n)
            if hi <= lo:
                continue
            page, i = int(s.table[b, t0 // s.ps]), t0 % s.ps // BLOCK
            rows = slice(at + lo - (n - m), at + hi - (n - m))
            for name, want, size in (("k", wk, sk), ("v", wv, None)):
                slack = 0.0
                for g in range(s.hkv):
                    y = want[rows, g]
                    if size is not None:
                        slack = SLACK * size[rows, g]
                    _check_block(s, name, *before[name], page, g, i, lo - t0, y, slack)
                touched[name][0][page, :, t0 % s.ps:t0 % s.ps + BLOCK] = True
                touched[name][1][page, :, i] = True
        at += m
    for name, codes, scale in (("k", s.k, s.k_scale), ("v", s.v, s.v_scale)):
        for now, was, mine in zip((codes, scale), before[name], touched[name]):
            assert bool(((u8(now) == was) | mine).all()), name
    return q


APPEND = {
    # name: (new tokens, lengths, query heads, KV heads, page, dtype, norms, layout)
    "one_token": ([1], [1], 4, 2, 16, BF, False, "plain"),
    "step_of_five": ([1] * 5, [33, 1, 16, 17, 250], 32, 8, 16, BF, False, "plain"),
    "step_fp16": ([1] * 4, [40, 64, 31, 9], 8, 4, 64, FP, True, "plain"),
    "prompts": ([40, 1, 65], [40, 1, 65], 8, 2, 32, FP, True, "plain"),
    "chunk_far_out": ([33], [100033], 4, 1, 128, FP, False, "plain"),
    "chunk_far_out_normed": ([20], [100033], 4, 1, 128, BF, True, "plain"),
    "drafts": ([5, 3, 9, 2], [21, 17, 40, 130], 14, 2, 32, BF, False, "plain"),
    "none_and_some": ([0, 3, 0, 0, 18, 0], [5, 3, 0, 31, 20, 7], 6, 3, 16, BF, True, "plain"),
    "heads_first": ([9, 2], [30, 50], 14, 2, 32, FP, True, "heads_first"),
    "pages_apart": ([9, 2], [30, 50], 8, 8, 64, BF, False, "apart"),
    "many_requests": ([1, 0, 2] * 70, [5, 9, 18] * 70, 2, 1, 16, BF, False, "plain"),
    "many_kv_heads": ([20], [25], 11, 11, 16, FP, False, "plain"),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(APPEND))
def test_append(dev, name):
    new, lens, hq, hkv, ps, dt, norms, layout = APPEND[name]
    print(f"[gpu] paged append8 {name}", flush=True)
    s = Step8(dev, new, lens, hkv=hkv, ps=ps, dtype=dt, layout=layout, seed=3, data=False)
    _check_append(s, hq, norms=norms)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("up", [-6, -1, 1, 2, 5])
def test_append_to_a_block_of_other_size(dev, dtype, up):
    """New tokens 2^up times as large as the earlier ones of their block: its scale stays, or rises and the
    earlier codes are rounded again, down to those that vanish."""
    print(f"[gpu] paged append8 up {up}", flush=True)
    s = Step8(dev, [2, 7, 1], [9, 25, 16], hkv=2, dtype=dtype, seed=31, data=False, spread=0, unit=-2)
    qkv = (s.rand(s.T, 8 * DH).float() * 2.0 ** up / 4).to(dtype)
    _check_append(s, 4, qkv=qkv)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_append_extreme_values(dev, dtype):
    """Values from the least to the largest of the type, ties between codes, zeros, one value alone; what
    is not finite is held as NaN and leaves the others' scale alone."""
    print("[gpu] paged append8 extremes", flush=True)
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    sizes = [big, big / 2, 1.0, 0.02, 2.0**-14, tiny * 4, tiny, tiny / 64, 0.0]
    hkv = len(sizes)
    s = Step8(dev, [16, 16, 3, 1], [16, 16, 3, 1], hkv=hkv, dtype=dtype, seed=33, data=False)
    qkv = s.rand(s.T, 3 * hkv * DH).float().view(s.T, 3, hkv, DH).clamp(-1, 1)
    qkv *= torch.tensor(sizes, dtype=torch.float64, device=dev)[None, None, :, None].float()
    # ties: every half step of e4m3 around a largest of 448
    half = torch.cat([GRID, (GRID[1:] + GRID[:-1]) / 2]).float().to(dev)
    qkv[:16, 2, 2] = 0.0
    qkv[:2, 2, 2] = half[:256 - 3].new_zeros(2 * DH).index_copy_(
        0, torch.arange(253, device=dev), half).view(2, DH)
    qkv[18, 2, 3], qkv[18, 2, 3, 5] = 0.0, -1.0
    qkv = qkv.clamp(-big, big).to(dtype).view(s.T, -1)
    _check_append(s, hkv, qkv=qkv)
    bad = qkv.view(s.T, 3, hkv, DH).clone()
    bad[3, 2, 2, 7], bad[4, 2, 2, 8], bad[20, 2, 1, 0] = math.inf, math.nan, -math.inf
    bad[5, 1, 2, 9], bad[6, 1, 3, 70] = math.inf, math.nan
    t = Step8(dev, [16, 16, 3, 1], [16, 16, 3, 1], hkv=hkv, dtype=dtype, seed=33, data=False)
    paged_append(bad.view(s.T, -1), t.k, t.v, t.batch, heads=hkv, theta=500000.0, **t.both)
    n = t.k.double().isnan()
    page = int(t.table[0, 0])
    for row, g, d in ((5, 2, (9, 73)), (6, 3, (6 + 64, 6))):
        assert sorted(torch.nonzero(n[page, g, row])[:, 0].tolist()) == sorted(d)
    v = t.v.double().isnan()[page]
    assert int(v.sum()) == 2 and bool(v[2, 3, 7]) and bool(v[2, 4, 8])
    for name in ("k", "v"):  # every other code as without them
        now, was = u8(getattr(t, name)), u8(getattr(s, name))
        same = (now == was) | getattr(t, name).double().isnan()
        assert bool(same.all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_append_keeps_earlier_nans(dev, dtype):
    """NaN codes of earlier tokens stay NaN where the block's scale rises; codes of both signs of zero and
    the largest are rounded again as the others are."""
    print("[gpu] paged append8 earlier NaN", flush=True)
    s = Step8(dev, [2, 1], [14, 9], hkv=2, dtype=dtype, seed=35, data=False, spread=0, unit=-1)
    page = int(s.table[0, 0])
    for t in (s.k, s.v):
        t.view(torch.uint8)[page, :, 3, :5] = torch.tensor([0x7f, 0xff, 0x80, 0x7e, 0xfe],
                                                           dtype=torch.uint8, device=dev)
    _check_append(s, 4, qkv=(s.rand(s.T, 8 * DH).float() * 8).to(dtype))
    assert s.v[page, 0, 3, :2].double().isnan().all()


@pytest.mark.gpu
def test_append_leaves_padding_rows_and_what_has_no_place(dev):
    """Rows behind the last request, tokens whose page is outside the pool or past the table."""
    print("[gpu] paged append8 padding, bad pages", flush=True)
    s = Step8(dev, [3, 0, 4], [20, 4, 4], hkv=2, seed=5, pad=30, data=False)
    out = torch.full((s.T, 4, DH), 7.0, dtype=BF, device=dev)
    _check_append(s, 4, out=out, norms=True)
    assert bool((out[s.rows:] == 7.0).all()) and not bool((out[:s.rows] == 7.0).all())
    s = Step8(dev, [20, 4, 3], [40, 4, 3], hkv=2, seed=6, data=False)
    u8k, u8s = u8(s.k).clone(), u8(s.k_scale).clone()
    table = s.table.clone()
    table[0, 1], table[1, 0] = -5, 2**30  # tokens 16 .. 31 of request 0, all of request 1
    lens = torch.tensor([40, 4, 2], dtype=torch.int32, device=dev)
    batch = PagedBatch(table.to(dev), s.batch.q_start, lens, rows=s.rows, max_new=20, max_len=40)
    qkv = s.rand(s.T, 8 * DH)
    q = paged_append(qkv, s.k, s.v, batch, heads=4, theta=1e4,
                     out=torch.zeros(s.T, 4, DH, dtype=BF, device=dev), **s.both)
    assert bool((q[24] == 0).all()) and bool((q[:24].abs().sum((1, 2)) > 0).all())
    page = int(s.table[0, 2])
    changed = (u8(s.k) != u8k).any(-1)  # (pages, heads, slots)
    want = torch.zeros_like(changed)
    want[page, :, :8] = True
    want[int(s.table[2, 0]), :, :2] = True
    assert torch.equal(changed, want)
    blocks = (u8(s.k_scale) != u8s)
    assert int(blocks.sum()) == 4
    cut = PagedBatch(s.table[:, :1].contiguous().to(dev), s.batch.q_start, s.batch.lens,
                     rows=s.rows, max_new=20, max_len=16)
    k0 = u8(s.k).clone()
    paged_append(qkv, s.k, s.v, cut, heads=4, theta=1e4, **s.both)
    assert bool(((u8(s.k) != k0).any(-1) <= (torch.zeros_like(want).index_fill_(
        0, s.table[1:3, 0].long().to(dev), True))).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_tokens_one_by_one_are_held_as_at_once(dev, dtype):
    """A prompt at once, in pieces and token by token: the same scales, and values that differ only where
    a code fell below the smallest normal one (rounded more than once there)."""
    print("[gpu] paged append8 pieces", flush=True)
    n, hkv = 50, 2
    g = torch.Generator().manual_seed(5)
    qkv = (torch.randn(n, 4 * hkv * DH, generator=g)
           * torch.exp2(torch.randint(-3, 4, (n, 1), generator=g).float())).to(dtype).to(dev)
    held = []
    for pieces in ([n], [7, 20, 1, 22], [1] * n):
        cache = PagedKVCache(1, 4, hkv, page_size=16, dtype=CODES, device=dev)
        r, at = cache.add(), 0
        for m in pieces:
            batch = cache.batch([(r, m)])
            paged_append(qkv[at:at + m], cache.k[0], cache.v[0], batch, heads=2 * hkv, theta=1e4,
                         k_scale=cache.k_scale[0], v_scale=cache.v_scale[0])
            at += m
        ids = torch.tensor(cache.page_ids(r), dtype=torch.int32, device=dev)
        k, v = paged_values(cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0], pages=ids,
                            dtype=torch.float32)
        at = ids.long()
        held.append([t.transpose(1, 2).reshape(-1, hkv, DH)[:n] for t in (k, v)]
                    + [u8(cache.k_scale[0])[at], u8(cache.v_scale[0])[at]])
    for other in held[1:]:
        for kind in (0, 1):
            e = held[0][2 + kind]
            assert torch.equal(other[2 + kind], e)
            step = two_to(e.long() - 127).float().repeat_interleave(16, 2).transpose(1, 2).reshape(
                -1, hkv, 1)[:n]
            a, b = other[kind], held[0][kind]
            # below 2^-6 of a scale codes are 2^-9 apart: rounded twice or more, a step at most
            assert bool(((a == b) | ((a.abs() <= step * 2.0**-6) & ((a - b).abs() <= step * 2.0**-9)))
                        .all())


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def _check_attend(s, hq, *, scale=None, qscale=1.0, q=None):
    if q is None:
        q = s.rand(s.T, hq, DH, scale=qscale)
    s.forget()
    want, tol = _attend_reference(s, q, scale)
    got = paged_attention(q, s.k, s.v, s.batch, scale=scale, out_dtype=torch.float32, **s.both)
    # Prompts' weights w_k are rounded once, to w_k (1 + d_k) with |d_k| at most half a step, and divided by
    # the sum of what they became: sum w_k (1 + d_k) v_k / sum w_k (1 + d_k) is off by sum p_k (d_k - d) v_k,
    # d the mean of the d_k: up to two half steps of sum p_k |v_k|, where the reference counts one.
    tol = 2 * tol
    err = (got[:s.rows].double() - want).abs()
    print(f"[gpu]   err/tol {float((err / (tol + 1e-30)).max()):.3f}", flush=True)
    good = bool((err <= tol + 1e-30).all())
    assert good
    got16 = paged_attention(q, s.k, s.v, s.batch, scale=scale, **s.both)
    assert got16.dtype == s.dtype and torch.equal(got16[:s.rows], got[:s.rows].to(s.dtype))
    return got


ATTEND = {
    # name: (new tokens, lengths, query heads, KV heads, page, dtype, layout)
    "one_key": ([1], [1], 4, 2, 16, BF, "plain"),
    "lens_around_tiles": ([1] * 10, [15, 16, 17, 31, 32, 33, 63, 64, 65, 129], 8, 2, 16, BF, "plain"),
    "step_fp16": ([1] * 5, [1, 300, 77, 1023, 512], 32, 8, 32, FP, "plain"),
    "step_long": ([1, 1], [8195, 5000], 32, 8, 64, BF, "plain"),
    "one_long": ([1], [20011], 8, 8, 128, FP, "plain"),
    "hpg16": ([1, 1, 1], [700, 31, 1500], 32, 2, 16, BF, "plain"),
    "hpg7_drafts": ([5, 2, 7], [500, 90, 7], 14, 2, 16, FP, "plain"),
    "drafts_long": ([4, 3], [6000, 4097], 8, 2, 32, BF, "plain"),
    "hpg3_prompt": ([100, 33], [100, 33], 6, 2, 16, BF, "plain"),
    "prompt": ([257, 64], [257, 64], 8, 2, 64, FP, "plain"),
    "prompt_odd": ([333, 1, 190], [333, 1, 190], 4, 4, 128, BF, "plain"),
    "prompt_wide": ([300] * 6, [300] * 6, 32, 8, 16, BF, "plain"),
    "chunk": ([130, 61], [1500, 61], 8, 2, 16, BF, "plain"),
    "chunk_long": ([40], [9001], 8, 2, 32, FP, "plain"),
    "chunk_longer": ([70, 500], [5007, 2100], 8, 4, 64, BF, "plain"),
    "mixed": ([1, 1, 150, 1, 0, 3, 1], [400, 17, 700, 1, 9, 2000, 64], 8, 2, 32, BF, "plain"),
    "heads_first": ([1, 70], [130, 95], 8, 2, 32, FP, "heads_first"),
    "pages_apart": ([1, 70, 2], [130, 95, 600], 16, 1, 16, BF, "apart"),
    "none_at_all": ([0, 2, 0], [5, 2, 0], 4, 1, 16, BF, "plain"),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(ATTEND))
def test_attention(dev, name):
    new, lens, hq, hkv, ps, dt, layout = ATTEND[name]
    print(f"[gpu] paged attention8 {name}", flush=True)
    _check_attend(Step8(dev, new, lens, hkv=hkv, ps=ps, dtype=dt, layout=layout, seed=11), hq)


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1, 1], [700, 90]), ([80, 5], [300, 200])])
def test_attention_peaked_and_scaled(dev, new, lens):
    """A near one-hot softmax (the running maximum rises late), and a scale of its own."""
    print(f"[gpu] paged attention8 peaked {new}", flush=True)
    _check_attend(Step8(dev, new, lens, hkv=2, seed=12), 8, qscale=8.0)
    _check_attend(Step8(dev, new, lens, hkv=2, seed=13, dtype=FP), 8, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("new,lens", [([1, 1], [700, 90]), ([80, 5], [300, 200])])
def test_attention_scales_far_apart(dev, new, lens, dtype):
    """Blocks whose scales differ by up to 2^14 (fp16) and 2^60 (bf16) in one tile, values that are large and
    tiny; keys small enough for the scores to stay moderate."""
    print(f"[gpu] paged attention8 scales {new}", flush=True)
    s = Step8(dev, new, lens, hkv=2, seed=14, dtype=dtype)
    g = torch.Generator().manual_seed(3)
    n = s.v_scale.numel()
    lo, hi = (-14, 0) if dtype == FP else (-60, 0)
    e = torch.randint(lo, hi + 1, (n,), generator=g) + 127
    s.v_scale.view(torch.uint8).copy_(e.to(torch.uint8).view(s.v_scale.shape))
    e = torch.randint(-14, -7, (n,), generator=g) + 127
    s.k_scale.view(torch.uint8).copy_(e.to(torch.uint8).view(s.k_scale.shape))
    _check_attend(s, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1] * 3, [700, 90, 33]), ([80, 5], [300, 200])])
def test_attention_leaves_padding_rows(dev, new, lens):
    print(f"[gpu] paged attention8 padding {new}", flush=True)
    s = Step8(dev, new, lens, hkv=2, seed=14, pad=9)
    q = s.rand(s.T, 8, DH)
    want, tol = _attend_reference(s, q)
    whole = torch.full((s.T, 9, 2 * DH), 3.0, dtype=torch.float32, device=dev)
    out = whole[:, :8, :DH]
    got = paged_attention(q, s.k, s.v, s.batch, out=out, **s.both)
    good = got.data_ptr() == out.data_ptr() and bool(
        ((out[:s.rows].double() - want).abs() <= 2 * tol + 1e-30).all())
    assert good
    out[:s.rows] = 3.0
    assert bool((whole == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 3, 60])
def test_attention_masks_pages_that_are_not_there(dev, new):
    """A page id outside the pool: its keys are masked, as if their tokens were others'. No page at all, or
    a length of zero: 0."""
    print(f"[gpu] paged attention8 bad pages {new}", flush=True)
    s = Step8(dev, [new] * 4, [150, 150, 150, 60], hkv=2, seed=15)
    q = s.rand(s.T, 4, DH)
    want, tol = _attend_reference(s, q)
    s.table[1, 2], s.table[1, 5] = -1, 10**6      # tokens 32 .. 47 and 80 .. 95 of request 1
    s.table[2] = -1                               # all of request 2
    lens = torch.tensor([150, 150, 150, 0], dtype=torch.int32, device=dev)
    batch = PagedBatch(s.table.to(dev), s.batch.q_start, lens, rows=s.rows, max_new=new,
                       max_len=150, min_new=new)
    got = paged_attention(q, s.k, s.v, batch, out_dtype=torch.float32, **s.both)
    pos = torch.arange(150 - new, 150, device=dev)[:, None]
    key = torch.arange(150, device=dev)[None]
    dead = (key > pos) | ((key // 16) == 2) | ((key // 16) == 5)
    good = [int(i) if 0 <= int(i) < s.k.shape[0] else 0 for i in s.table[1, :10]]
    k_all, v_all = s.held(s.k).nan_to_num(), s.held(s.v).nan_to_num()
    for h in range(4):
        k, v = (t[good, h // 2].reshape(-1, DH)[:150] for t in (k_all, v_all))
        z = (q[new:2 * new, h].double() @ k.T / math.sqrt(DH)).masked_fill(dead, -math.inf)
        p = torch.softmax(z, -1)
        # the weights' two half steps and fp32 scores of up to 2^6: 2^-7 covers both
        fine = (got[new:2 * new, h].double() - p @ v).abs() <= 2.0**-7 * (p @ v.abs()) + 1e-30
        assert bool(fine.all())
    first = bool(((got[:new].double() - want[:new]).abs() <= 2 * tol[:new] + 1e-30).all())
    assert first and bool((got[2 * new:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new,n,hkv", [(4, 300, 2), (60, 60, 2), (60, 3000, 2), (700, 700, 8)])
def test_attention_keeps_later_tokens_out(dev, new, n, hkv):
    """A NaN in a new token's value or key: the tokens before it have the result they have without it; the
    ones from it on have it in theirs."""
    print(f"[gpu] paged attention8 later {new}", flush=True)
    s = Step8(dev, [new, 1], [n, 40], hkv=hkv, seed=17)
    q = s.rand(s.T, 4 * hkv, DH)
    attend = lambda: paged_attention(q, s.k, s.v, s.batch, out_dtype=torch.float32, **s.both)  # noqa: E731
    clean = attend()
    _, tol = _attend_reference(s, q)
    bad = n - new + new // 2  # the position of the token
    page, slot = int(s.table[0, bad // 16]), bad % 16
    before, after = slice(0, new // 2), slice(new // 2, new)
    s.v.view(torch.uint8)[page, :, slot, ::3] = 0xff
    got = attend()
    near = lambda a, b, t: bool(((a - b).abs() <= 4 * t).all())  # noqa: E731
    assert near(got[before], clean[before], tol[before]) and torch.equal(got[new:], clean[new:])
    assert bool(got[after][..., ::3].isnan().all())
    assert near(got[after][..., 1::3], clean[after][..., 1::3], tol[after][..., 1::3])
    s.k.view(torch.uint8)[page, :, slot] = 0x7f
    got = attend()
    assert near(got[before], clean[before], tol[before]) and torch.equal(got[new:], clean[new:])
    assert bool(got[after].isnan().all())


def _random_step(i):
    g = torch.Generator().manual_seed(900 + i)
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
    print(f"[gpu] random step8 {i}: {new} {lens} {hq}/{hkv} page {ps} {dt}", flush=True)
    s = Step8(dev, new, lens, hkv=hkv, ps=ps, dtype=dt, seed=600 + i)
    q = _check_append(s, hq, norms=i % 2 == 0)
    _check_attend(s, hq, q=q)


MANY = {
    # more units than workgroups of eight waves, of four, and requests than a wave holds the lengths of
    "four_waves": ([1] * 35, [40, 3000, 7, 500, 64] * 7, 32, 8, 16),
    "uncut": ([1] * 70, [40, 300, 7, 500, 64] * 14, 32, 8, 16),
    "many_requests": ([1, 1, 0] * 100, [40, 300, 7] * 100, 8, 2, 16),
    "many_requests_one_head": ([1] * 400, [40, 300] * 200, 4, 1, 32),
    "with_prompts": ([1, 1, 40] * 30, [40, 300, 47] * 30, 8, 2, 16),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(MANY))
def test_attention_many_requests(dev, name):
    new, lens, hq, hkv, ps = MANY[name]
    print(f"[gpu] paged attention8 many {name}", flush=True)
    s = Step8(dev, new, lens, hkv=hkv, ps=ps, seed=51)
    q = s.rand(s.T, hq, DH)
    got = paged_attention(q, s.k, s.v, s.batch, out_dtype=torch.float32, **s.both)
    hpg = hq // hkv
    k_all, v_all = s.held(s.k), s.held(s.v)
    for b, (m, n) in enumerate(zip(new, lens)):
        if m == 0:
            continue
        ids = s.table[b, :-(-n // ps)].long().to(dev)
        k, v = (t[ids].transpose(0, 1).reshape(hkv, -1, DH)[:, :n].repeat_interleave(hpg, 0)
                for t in (k_all, v_all))
        x = q[s.starts[b]:s.starts[b] + m].double().transpose(0, 1)
        z = torch.matmul(x, k.transpose(1, 2).contiguous()) / math.sqrt(DH)
        z.masked_fill_(torch.arange(n, device=dev)[None] > torch.arange(n - m, n, device=dev)[:, None],
                       -math.inf)
        p = torch.softmax(z, -1)
        want, size = torch.matmul(p, v).transpose(0, 1), torch.matmul(p, v.abs()).transpose(0, 1)
        # two half steps of the weights, and fp32 scores: 2^-7 covers both
        fine = (got[s.starts[b]:s.starts[b] + m].double() - want).abs() <= 2.0**-7 * size + 1e-30
        assert bool(fine.all()), (b, m, n)


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_requests_that_come_and_go(dev, dtype):
    """Three requests through a cache: prompts in chunks beside single tokens, one ended and its pages
    reused, one cut back; every output against attention over the values that the pages hold, and these
    against the tokens kept aside, half a step of e4m3 (2^-4, or 2^-10 of a block's scale) away."""
    print("[gpu] paged8 chunks", flush=True)
    hq, hkv, theta = 8, 2, 10000.0
    cache = PagedKVCache(1, 24, hkv, page_size=16, dtype=CODES, device=dev)
    cache.k[0].view(torch.uint8).fill_(0x7f), cache.v[0].view(torch.uint8).fill_(0x7f)
    g = torch.Generator().manual_seed(77)
    both = dict(k_scale=cache.k_scale[0], v_scale=cache.v_scale[0])
    kept: dict = {}
    a, b, c = cache.add(), cache.add(), cache.add()

    def step(parts):
        qkv = torch.randn(sum(n for _, n in parts), (hq + 2 * hkv) * DH, generator=g).to(dtype).to(dev)
        batch = cache.batch(parts)
        q = paged_append(qkv, cache.k[0], cache.v[0], batch, heads=hq, theta=theta, **both)
        o = paged_attention(q, cache.k[0], cache.v[0], batch, out_dtype=torch.float32, **both)
        at = 0
        for r, n in parts:
            kept[r] = torch.cat([kept[r], qkv[at:at + n]]) if r in kept else qkv[at:at + n]
            total = kept[r].shape[0]
            assert total == cache.length(r)
            ids = torch.tensor(cache.page_ids(r), dtype=torch.int32, device=dev)
            held = paged_values(cache.k[0], cache.v[0], **both, pages=ids, dtype=torch.float32)
            k, v = (t.transpose(1, 2).reshape(-1, hkv, DH)[:total].double() for t in held)
            x = kept[r].double().view(total, hq + 2 * hkv, DH)
            pos = torch.arange(total, dtype=torch.float64, device=dev)
            for got, want, scale in ((k, _turn(x[:, hq:hq + hkv], pos, _freq(dev, theta)), 0),
                                     (v, x[:, hq + hkv:], 1)):
                e = u8(cache.v_scale[0] if scale else cache.k_scale[0])[ids.long()].double() - 127
                two = two_to(e).repeat_interleave(16, 2).transpose(1, 2).reshape(-1, hkv, 1)[:total]
                # (once more where a block's scale rose later: two roundings below the normal codes)
                fine = (got - want).abs() <= 2.0**-4 * want.abs() + 2 * 2.0**-10 * two
                assert bool(fine.all())
            for h in range(hq):
                z = q[at:at + n, h].double() @ k[:, h // 4].T / math.sqrt(DH)
                z.masked_fill_(torch.arange(total, device=dev)[None]
                               > torch.arange(total - n, total, device=dev)[:, None], -math.inf)
                p = torch.softmax(z, -1)
                fine = ((o[at:at + n, h].double() - p @ v[:, h // 4]).abs()
                        <= 2.0**-7 * (p @ v[:, h // 4].abs()) + 1e-30)
                assert bool(fine.all()), (r, total, h)
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
    """A captured append, attention and reading back, replayed with other inputs, lengths and pages in the
    same buffers, with eager work between the replays; two graphs replayed at once on two streams."""
    print(f"[gpu] paged8 graph {new}", flush=True)
    side = torch.cuda.Stream()
    s = [Step8(dev, new, lens, hkv=2, seed=21 + i) for i in range(2)]
    qkv = [t.rand(t.T, 12 * DH) for t in s]

    def one(i):
        t = s[i]
        q = paged_append(qkv[i], t.k, t.v, t.batch, heads=8, theta=1e4, **t.both)
        return (paged_attention(q, t.k, t.v, t.batch, **t.both),
                *paged_values(t.k, t.v, **t.both, pages=t.batch.page_table.view(-1)))

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
    other = Step8(dev, [1], [3000], hkv=2, seed=29)
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
        paged_attention(oq, other.k, other.v, other.batch, **other.both)
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for i in range(2):
            t = s[i]
            got = [u8(x).clone() for x in (*outs[i], t.k, t.v, t.k_scale, t.v_scale)]
            again = one(i)
            for x, y in zip(got, (*again, t.k, t.v, t.k_scale, t.v_scale)):
                assert torch.equal(x, u8(y)), (rep, i)


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    print("[gpu] paged8 two streams", flush=True)
    s = [Step8(dev, [1, 2], [1500, 1100 + 300 * i], hkv=2, seed=31 + i) for i in range(2)]
    q = [t.rand(t.T, 8, DH) for t in s]
    run = lambda i: paged_attention(q[i], s[i].k, s[i].v, s[i].batch, **s[i].both)  # noqa: E731
    want = [run(i) for i in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


@pytest.mark.gpu
def test_pool_past_32_bits(dev):
    """Pages whose codes lie past 2^32 bytes of the pool's start."""
    print("[gpu] paged8 large pool", flush=True)
    ps, hkv, pages = 256, 2, 70000  # 4.6 GB each for keys and values
    k = torch.empty(pages, hkv, ps, DH, dtype=torch.uint8, device=dev).view(CODES)
    v = torch.empty_like(k)
    ks = torch.zeros(pages, hkv, ps // 16, dtype=torch.uint8, device=dev).view(SCALES)
    vs = torch.zeros_like(ks)
    for new, n in ((1, 700), (70, 700)):
        ids = [pages - 1, 3, pages - 900]
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        batch = PagedBatch(i32(*ids)[None], i32(0, new), i32(n), rows=new, max_new=new, max_len=n,
                           min_new=new)
        small = Step8(dev, [new], [n], hkv=hkv, ps=ps, seed=42)
        qkv = small.rand(new, 8 * DH)
        order = small.table[0, :3].long().to(dev)
        for big, part in ((k, small.k), (v, small.v), (ks, small.k_scale), (vs, small.v_scale)):
            big.view(torch.uint8)[ids] = part.view(torch.uint8)[order]
        both = dict(k_scale=ks, v_scale=vs)
        qa = paged_append(qkv, k, v, batch, heads=4, theta=1e4, **both)
        qb = paged_append(qkv, small.k, small.v, small.batch, heads=4, theta=1e4, **small.both)
        assert torch.equal(qa, qb)
        for big, part in ((k, small.k), (v, small.v), (ks, small.k_scale), (vs, small.v_scale)):
            assert torch.equal(big.view(torch.uint8)[ids], part.view(torch.uint8)[order])
        assert torch.equal(paged_attention(qa, k, v, batch, **both),
                           paged_attention(qb, small.k, small.v, small.batch, **small.both))
        a = paged_values(k, v, **both, pages=i32(*ids))
        b = paged_values(small.k, small.v, **small.both, pages=order.int())
        assert torch.equal(u8(a[0]), u8(b[0])) and torch.equal(u8(a[1]), u8(b[1]))


# ---------------------------------------------------------------------------------------------
# pages read back
# ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP, torch.float32])
@pytest.mark.parametrize("layout,ps,hkv", [("plain", 16, 1), ("heads_first", 32, 3), ("apart", 64, 2)])
def test_values(dev, dtype, layout, ps, hkv):
    """Every code under scales from the least to the largest that an append gives; NaN codes and scales;
    chosen pages, some of them outside the pool; a page twice; none."""
    print(f"[gpu] paged values {layout} {dtype}", flush=True)
    s = Step8(dev, [1], [1], ps=ps, hkv=hkv, spare=9, layout=layout, data=False, seed=1)
    g = torch.Generator().manual_seed(9)
    s.k.view(torch.uint8).copy_(torch.randint(0, 256, s.k.shape, generator=g, dtype=torch.uint8))
    s.v.view(torch.uint8).copy_(torch.randint(0, 256, s.v.shape, generator=g, dtype=torch.uint8))
    low, high = RANGE.get(dtype, (-110, 119))
    for t in (s.k_scale, s.v_scale):
        e = torch.randint(low, high + 1, t.shape, generator=g) + 127
        t.view(torch.uint8).copy_(e.to(torch.uint8))
        t.view(torch.uint8)[2, 0, 0] = 255
    same = lambda a, b: bool(((a.double() == b) | (a.isnan() & b.isnan())).all())  # noqa: E731
    k, v = paged_values(s.k, s.v, **s.both, dtype=dtype)
    assert k.dtype == dtype and k.is_contiguous() and k.shape == s.k.shape
    assert same(k, s.held(s.k)) and same(v, s.held(s.v))
    ids = torch.tensor([4, -1, 0, 4, s.k.shape[0], 2**30], dtype=torch.int32, device=dev)
    k, v = paged_values(s.k, s.v, **s.both, pages=ids, dtype=dtype)
    for got, whole in ((k, s.held(s.k)), (v, s.held(s.v))):
        assert got.shape[0] == 6 and not bool(got[[1, 4, 5]].any())
        assert same(got[[0, 2, 3]], whole[[4, 0, 4]])
    k, v = paged_values(s.k, s.v, **s.both, pages=ids[:0], dtype=dtype)
    assert k.shape == (0, hkv, ps, DH) and v.shape == k.shape


@pytest.mark.gpu
def test_same_with_and_without_the_tensor_module(dev, monkeypatch):
    from dynakv_amd import _lib
    print("[gpu] paged8 without the tensor module", flush=True)
    out = []
    for off in (False, True):
        if off:
            monkeypatch.setattr(_lib, "_tensor_calls", None)
        got = []
        for new, lens, dt in (([1, 1], [30, 2000], BF), ([70, 3], [100, 90], FP)):
            s = Step8(dev, new, lens, hkv=2, seed=61, dtype=dt)
            qkv = s.rand(s.T, 12 * DH)
            q = paged_append(qkv, s.k, s.v, s.batch, heads=8, theta=1e4, **s.both)
            got += [q, paged_attention(q, s.k, s.v, s.batch, **s.both), s.k, s.v, s.k_scale, s.v_scale]
            got += paged_values(s.k, s.v, **s.both, dtype=dt)
            got += paged_values(s.k, s.v, **s.both, pages=s.batch.page_table[0], dtype=torch.float32)
        out.append(got)
    for x, y in zip(*out):
        assert x.dtype == y.dtype and torch.equal(u8(x), u8(y))
