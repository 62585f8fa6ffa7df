"""The append to 8-bit pages of many requests in one call: what calls of 64 requests each leave, to the bit."""
import pytest
import torch

from dynakv_amd.kernels.paged import PagedBatch, paged_append

DH, HKV, HQ, PS = 128, 2, 4, 32
CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _some(n, lo, hi, seed):
    return torch.randint(lo, hi, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


CASES = {
    # name: (new tokens, rows before the first request, rows behind the last)
    "single_tokens_257": ([1] * 257, 0, 0),
    "single_tokens_5000": ([1] * 5000, 0, 3),
    "one_or_none_4097": (_some(4097, 0, 2, 1), 5, 0),
    "drafts_700": (_some(700, 0, 5, 2), 0, 40),
    "chunks_270": (_some(270, 0, 61, 3), 0, 0),
    "chunks_300": ([40] * 300, 17, 9),
    "two_prompts_beside_300": ([1] * 60 + [700] + [0] * 120 + [650] + [2] * 118, 0, 0),
    "idle_requests_3000": ([0] * 1500 + [33, 1, 16] + [0] * 1497, 0, 1),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", list(CASES))
def test_as_calls_of_64_requests(dev, name, dtype):
    """Positions anywhere in their blocks; earlier tokens in them; some requests whose pages or lengths do not
    hold their tokens, whose table ends before them or who have fewer tokens than rows."""
    print(f"[gpu] paged append8 requests {name} {dtype}", flush=True)
    new, head, tail = CASES[name]
    B, g = len(new), torch.Generator().manual_seed(9)
    earlier = torch.randint(0, 50, (B,), generator=g).tolist()
    lens = [n + e for n, e in zip(new, earlier)]
    cols = max(-(-n // PS) for n in lens)
    pages = sum(-(-n // PS) for n in lens) + 1
    ids = torch.randperm(pages, generator=g).to(torch.int32)
    table, at = torch.full((B, cols), -1, dtype=torch.int32), 0
    for b, n in enumerate(lens):
        k = -(-n // PS)
        table[b, :k] = ids[at:at + k]
        at += k
    for b in range(11, B, 37):
        if b % 2:
            table[b, 0] = [-3, pages + 5][b % 3 == 0]   # no such page
        else:
            lens[b] = max(0, new[b] - 1)                # a row without a place
    starts = [head]
    for n in new:
        starts.append(starts[-1] + n)
    rows = starts[-1] + tail
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    qkv = (torch.randn(rows, (HQ + 2 * HKV) * DH, generator=g) * torch.exp2(
        torch.randint(-3, 4, (rows, 1), generator=g).float())).to(dtype).to(dev)
    kn = (1 + 0.2 * torch.randn(DH, generator=g)).to(dtype).to(dev)
    codes = torch.randint(0, 127, (2, pages, HKV, PS, DH), generator=g, dtype=torch.uint8).to(dev)
    scales = torch.randint(116, 124, (2, pages, HKV, PS // 16), generator=g, dtype=torch.uint8).to(dev)

    def pools():
        k, v = codes.clone().view(CODES).unbind()
        ks, vs = scales.clone().view(SCALES).unbind()
        return (k, v), dict(k_scale=ks, v_scale=vs)

    def call(lo, hi, pool, both, out, cut):
        batch = PagedBatch(table[lo:hi, :cut].contiguous().to(dev), i32(starts[lo:hi + 1]), i32(lens[lo:hi]),
                           rows=rows, max_new=rows, max_len=0)
        paged_append(qkv, *pool, batch, heads=HQ, theta=1e4, k_norm=kn, out=out, **both)

    for cut in (cols, max(1, cols // 2)):
        (a, both_a), (b, both_b) = pools(), pools()
        qa, qb = (torch.full((rows, HQ, DH), 9.0, dtype=dtype, device=dev) for _ in range(2))
        call(0, B, a, both_a, qa, cut)
        for lo in range(0, B, 64):
            call(lo, min(B, lo + 64), b, both_b, qb, cut)
        assert torch.equal(qa, qb)
        for x, y in zip((*a, *both_a.values()), (*b, *both_b.values())):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert not torch.equal(a[0].view(torch.uint8), codes[0])
