"""Indexes of pages read back that pass 32 bits: the split of a piece's number on the host, and a call of more
than 2^31 pieces on the GPU."""
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from dynakv_amd.kernels.paged import PagedBatch, paged_attention, paged_values

CSRC = Path(__file__).resolve().parent.parent / "dynakv_amd" / "csrc"
CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu

_MAIN = r"""
#include <cstdio>
#include "dkv_paged_index.h"
int main() {
  long long at;
  int shift;
  while (scanf("%lld %d", &at, &shift) == 2) {
    const PagedPiece a = paged_piece<16>(at, shift), b = paged_piece<32>(at, shift);
    printf("%d %d %d %d %d %d\n", a.row, a.slot, a.piece, b.row, b.slot, b.piece);
  }
}
"""

_SLOTS = r"""
#include <cstdio>
#include "dkv_paged_index.h"
int main() {
  int slot;
  while (scanf("%d", &slot) == 1) printf("%lld\n", paged_slot_at(slot));
}
"""


def _answers(tmp_path, source, text):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    (tmp_path / "main.cpp").write_text(source)
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(tmp_path / "main.cpp"), "-o",
                    str(tmp_path / "main")], check=True)
    return subprocess.run([str(tmp_path / "main")], input=text, capture_output=True, text=True,
                          check=True).stdout.split()


def test_slots_of_large_pages(tmp_path):
    """A slot's place in pages of 2^24 tokens and more."""
    slots = [0, 1, 2**24 - 1, 2**24, 2**24 + 5, 2**25 - 1, 2**25, 2**29 + 7]
    assert list(map(int, _answers(tmp_path, _SLOTS, " ".join(map(str, slots))))) == [
        128 * s for s in slots]


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 70, 1100])
def test_a_page_of_many_tokens(dev, new):
    """A page of 2^25 tokens, some of them past 2^31 elements of it: attention over it, in 8 and in 16 bits, and
    its values are those of the same memory as pages of 64 tokens."""
    print(f"[gpu] paged page of 2^25 tokens, {new} new", flush=True)
    n, whole = 2**24 + 900, 2**25
    g = torch.Generator(device=dev).manual_seed(6)
    pools, i32 = [], lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for _ in range(2):
        codes = torch.zeros(whole, 128, dtype=torch.uint8, device=dev)
        scales = torch.zeros(whole // 16, dtype=torch.uint8, device=dev)
        for lo, hi in ((0, 3000), (n - 2000, n)):  # the others' keys and values are 0
            codes[lo:hi].random_(0, 127, generator=g)
        scales.random_(116, 119, generator=g)
        pools.append((codes.view(CODES), scales.view(SCALES)))
    q = torch.randn(new, 4, 128, generator=g, device=dev).bfloat16()
    got = []
    for ps in (whole, 64):
        k, v = (c.view(whole // ps, 1, ps, 128) for c, _ in pools)
        ks, vs = (c.view(whole // ps, 1, ps // 16) for _, c in pools)
        table = torch.arange(whole // ps, dtype=torch.int32, device=dev)[None]
        batch = PagedBatch(table, i32(0, new), i32(n), rows=new, max_new=new, max_len=n, min_new=new)
        o = paged_attention(q, k, v, batch, k_scale=ks, v_scale=vs)
        k, v = paged_values(k, v, ks, vs)
        part = [t.view(whole, 128)[n - 2000:n].clone() for t in (k, v)]
        got.append((o, paged_attention(q, k, v, batch), *part))
        del k, v
    assert all(bool(o.any()) and not bool(o.isnan().any()) for o in got[0])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_split_of_a_piece(tmp_path):
    """Row, slot and piece of numbers on both sides of 2^31, 2^32 and 2^33, in Python's whole numbers."""
    cases = [(edge + d, shift) for edge in (64, 2**31, 2**32, 2**33, 3 * 2**32)
             for d in (-33, -32, -17, -16, -1, 0, 1, 5, 15, 16, 31, 32, 100) for shift in (4, 6, 12)]
    out = _answers(tmp_path, _MAIN, "".join(f"{a} {s}\n" for a, s in cases))
    got = [list(map(int, out[i:i + 6])) for i in range(0, len(out), 6)]
    assert len(got) == len(cases)
    for (at, shift), g in zip(cases, got):
        want = []
        for pieces in (16, 32):
            token, piece = divmod(at, pieces)
            want += [token >> shift, token & ((1 << shift) - 1), piece]
        assert g == want, (at, shift)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_of_more_pieces_than_31_bits(dev, dtype):
    """A small pool's pages, many times each: results of 34 GB, 16 bytes a piece, whose last pages' pieces are
    numbered past 2^31."""
    print(f"[gpu] paged values of 2^31 pieces {dtype}", flush=True)
    pool, hkv, ps = 64, 8, 256
    page_bytes = hkv * ps * 128 * (2 if dtype == torch.bfloat16 else 4)
    n = 2**31 * 16 // page_bytes + 300
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(dev)[0] < 2 * n * page_bytes + 2**33:
        pytest.skip("not enough free memory")
    g = torch.Generator().manual_seed(5)
    byte = lambda *d, lo=0, hi=127: torch.randint(lo, hi, d, generator=g, dtype=torch.uint8).to(dev)  # noqa: E731
    k, v = (byte(pool, hkv, ps, 128).view(CODES) for _ in range(2))
    ks, vs = (byte(pool, hkv, ps // 16, lo=117, hi=130).view(SCALES) for _ in range(2))
    whole = paged_values(k, v, ks, vs, dtype=dtype)
    ids = torch.randint(0, pool, (n,), generator=g).to(torch.int32).to(dev)
    out = paged_values(k, v, ks, vs, pages=ids, dtype=dtype)
    edge = n - 300  # its first piece is number 2^31
    for got, held in zip(out, whole):
        for a, b in ((0, 200), (edge - 200, edge), (edge, edge + 1), (edge + 1, n)):
            assert torch.equal(got[a:b], held[ids[a:b].long()]), (a, b)
    del out
    torch.cuda.empty_cache()


_BLOCKS = r"""
#include <cstdio>
#include "dkv_paged_index.h"
int main() {
  int start, b;
  while (scanf("%d %d", &start, &b) == 2) printf("%d\n", paged_block_place(start, b));
}
"""


def test_places_of_blocks(tmp_path):
    """A request has a place for every block that its new tokens can touch, wherever its rows and its tokens
    begin, and all of them fit the launch: rows / 16 + 2 for each request."""
    g = torch.Generator().manual_seed(4)
    starts = [0]
    for n in torch.cat([torch.randint(0, 70, (500,), generator=g), torch.arange(0, 70)]).tolist():
        starts.append(starts[-1] + n)
    out = list(map(int, _answers(tmp_path, _BLOCKS, "".join(f"{s} {b}\n" for b, s in enumerate(starts)))))
    for b in range(len(starts) - 1):
        n = starts[b + 1] - starts[b]
        most = max((pos + n - 1) // 16 - pos // 16 + 1 for pos in range(16)) if n else 0
        assert out[b + 1] - out[b] >= most, b
    assert out[0] == 0 and out[-1] == starts[-1] // 16 + 2 * (len(starts) - 1)
