"""Single and drafted tokens over pages: their weights go to the products as hi and lo parts, so that a
result is as near as fp32 sums are, not half a step of the 16-bit type away.

Keys and queries are small whole numbers (times a power of two), whose products and sums are exact: what
is left of a score's error is its product with the scale and a subtraction. The bound counts 2^-24 for each
rounding in fp32, relative to sum p |v|; ``Z`` is the largest score in log2 units:

* a weight: the scale (its constant and the product: 2 Z), the subtraction (up to 2 Z), times ln 2 < 1, and
  the exponential's instruction (4 are taken); a reference that is raised, at most Z + 1 times (a step is 3
  at least), multiplies by one more such exponential. Of the numerator and of the sum that divides it: twice;
* sums: a product of 32 numbers counts as 32 roundings, and a wave has at most ceil(n / 64) tiles of them
  (four waves, tiles of 16 tokens): 64 for every 128 keys; the waves' and the parts' joins and the
  division: 64;
* parts: bf16 hi + lo leave 2^-18 of a weight; fp16 2^-22, or 2^-25 where the weights' largest is 2^12: of
  n weights n 2^-37 of the largest value.

A result whose lo parts were lost lies outside the bound (``test_a_lost_part_would_show``)."""
import pytest
import torch

BF, FP = torch.bfloat16, torch.float16
DH = 128
SCALE = 0.5
CASES = {
    # name: (new tokens, lengths, query heads, KV heads, page size)
    "short": ([1] * 6, [3, 17, 33, 64, 100, 250], 8, 2, 16),
    "parts": ([1, 1], [2100, 1300], 8, 2, 64),
    "drafts": ([4, 3, 2], [300, 40, 9], 8, 2, 32),
    "drafts_of_five_heads": ([3, 3], [200, 77], 10, 2, 16),
    "four_waves": ([1] * 35, [40, 600, 7, 500, 64] * 7, 32, 8, 16),
    "uncut": ([1] * 70, [40, 300, 7, 500, 64] * 14, 16, 8, 16),
    "many_requests_one_head": ([1] * 300, [40, 300] * 150, 4, 1, 32),
    "beside_a_prompt": ([1, 4, 40], [300, 200, 47], 8, 2, 16),
}


class _Inputs:
    """Pools, table and queries of a case, on the host."""

    def __init__(self, name, dtype):
        self.new, self.lens, self.hq, self.hkv, self.ps = CASES[name]
        self.dtype = dtype
        g = torch.Generator().manual_seed(3 + len(name))
        need = [-(-n // self.ps) for n in self.lens]
        self.table = torch.full((len(need), max(need)), -1, dtype=torch.int32)
        ids, at = torch.randperm(sum(need), generator=g).to(torch.int32), 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        dims = (sum(need), self.hkv, self.ps, DH)
        whole = lambda lo, hi, *d: torch.randint(lo, hi + 1, d, generator=g)  # noqa: E731
        self.k = whole(-8, 8, *dims).float().to(torch.float8_e4m3fn)
        self.v = (torch.randn(*dims, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        blocks = (dims[0], self.hkv, self.ps // 16)
        self.k_scale = torch.full(blocks, 127 - 5, dtype=torch.uint8)
        self.v_scale = (whole(-2, 2, *blocks) + 127 - 7).to(torch.uint8)
        self.starts = [0]
        for n in self.new:
            self.starts.append(self.starts[-1] + n)
        self.q = whole(-4, 4, self.starts[-1], self.hq, DH).to(dtype)

    def values(self, codes, scale):
        two = torch.ldexp(torch.ones(scale.shape, dtype=torch.float64), scale.int() - 127)
        return codes.double() * two.repeat_interleave(16, -1)[..., None]

    def results(self):
        """(rows of single and drafted tokens, exact results, bounds, results without the lo parts)."""
        k_all, v_all = self.values(self.k, self.k_scale), self.values(self.v, self.v_scale)
        hpg, rows, out = self.hq // self.hkv, [], []
        for b, (m, n) in enumerate(zip(self.new, self.lens)):
            if m * hpg > 16:
                continue
            r = slice(self.starts[b], self.starts[b] + m)
            rows += range(r.start, r.stop)
            ids = self.table[b, :-(-n // self.ps)].long()
            k, v = (t[ids].transpose(0, 1).reshape(self.hkv, -1, DH)[:, :n].repeat_interleave(hpg, 0)
                    for t in (k_all, v_all))
            z = self.q[r].double().transpose(0, 1) @ k.transpose(1, 2) * SCALE / torch.log(
                torch.tensor(2.0, dtype=torch.float64))  # (hq, m, n)
            z.masked_fill_(torch.arange(n)[None] > torch.arange(n - m, n)[:, None], -torch.inf)
            w = torch.exp2(z - z.amax(-1, keepdim=True))
            total = w.sum(-1, keepdim=True)
            size = w @ v.abs() / total
            Z = z[z > -torch.inf].abs().max()
            count = 2 * (4 * Z + 4 * (Z + 2)) + 64 * -(-n // 128) + 64
            tol = size * (count * 2.0**-24 + (2.0**-18 if self.dtype == BF else 2.0**-22))
            if self.dtype == FP:
                tol = tol + n * 2.0**-37 * v.abs().max()
            lost = (w.to(self.dtype) if self.dtype == BF else (w * 2.0**12).to(self.dtype).double()
                    * 2.0**-12).double() @ v / total
            out.append([t.transpose(0, 1) for t in (w @ v / total, tol, lost)])
        return rows, *(torch.cat(t) for t in zip(*out))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("name", list(CASES))
def test_a_lost_part_would_show(name, dtype):
    _, want, tol, lost = _Inputs(name, dtype).results()
    assert float(((lost - want).abs() / tol).max()) > (4 if dtype == BF else 1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("name", list(CASES))
def test_single_tokens_keep_both_parts(dev, name, dtype):
    """Over 8-bit pages, and over 16-bit ones of the same values."""
    from dynakv_amd.kernels.paged import PagedBatch, paged_attention, paged_values
    print(f"[gpu] paged weights {name} {dtype}", flush=True)
    s = _Inputs(name, dtype)
    rows, want, tol, _ = s.results()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    batch = PagedBatch(s.table.to(dev), i32(s.starts), i32(s.lens), rows=s.starts[-1], max_new=max(s.new),
                       max_len=max(s.lens), min_new=min(s.new))
    k, v, q = s.k.to(dev), s.v.to(dev), s.q.to(dev)
    both = dict(k_scale=s.k_scale.to(dev).view(torch.float8_e8m0fnu),
                v_scale=s.v_scale.to(dev).view(torch.float8_e8m0fnu))
    coded = paged_attention(q, k, v, batch, scale=SCALE, out_dtype=torch.float32, **both)
    k16, v16 = paged_values(k, v, **both, dtype=dtype)
    plain = paged_attention(q, k16, v16, batch, scale=SCALE, out_dtype=torch.float32)
    for kind, got in (("codes", coded), ("16 bits", plain)):
        err = (got.cpu()[rows].double() - want).abs() / tol
        print(f"[gpu]   {kind}: err/tol {float(err.max()):.3f}", flush=True)
        assert bool((err <= 1).all()), kind


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("new,lens,hq,hkv", [([512] * 4, [512] * 4, 32, 8), ([1100], [1100], 32, 8),
                                             ([130, 61], [2500, 700], 8, 2), ([1, 1], [9000, 5000], 8, 2),
                                             ([1, 70, 3, 1], [600, 900, 300, 40], 8, 2)])
def test_same_bits_every_time(dev, new, lens, hq, hkv, dtype):
    """Prompts, chunks in key ranges, single tokens in parts, both kinds: calls on the same inputs, other
    work between them, have the same bits."""
    from dynakv_amd.kernels.paged import paged_attention
    from test_gpu_paged8 import Step8
    print(f"[gpu] paged8 again {new} {dtype}", flush=True)
    s, other = (Step8(dev, new, lens, hkv=hkv, ps=32, dtype=dtype, seed=71 + i) for i in range(2))
    q, p = s.rand(s.T, hq, DH), other.rand(s.T, hq, DH)
    first = paged_attention(q, s.k, s.v, s.batch, **s.both)
    assert not bool(first.isnan().any())
    for _ in range(8):
        paged_attention(p, other.k, other.v, other.batch, **other.both)
        assert torch.equal(paged_attention(q, s.k, s.v, s.batch, **s.both), first)
