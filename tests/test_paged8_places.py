"""Indexes of pages read back that pass 32 bits: the split of a piece's number on the host, and a call of more
than 2^31 pieces on the GPU."""
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from dynakv_amd.kernels.paged import paged_values

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


def test_split_of_a_piece(tmp_path):
    """Row, slot and piece of numbers on both sides of 2^31, 2^32 and 2^33, in Python's whole numbers."""
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    (tmp_path / "split.cpp").write_text(_MAIN)
    exe = tmp_path / "split"
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(tmp_path / "split.cpp"), "-o", str(exe)],
                   check=True)
    cases = [(edge + d, shift) for edge in (64, 2**31, 2**32, 2**33, 3 * 2**32)
             for d in (-33, -32, -17, -16, -1, 0, 1, 5, 15, 16, 31, 32, 100) for shift in (4, 6, 12)]
    out = subprocess.run([str(exe)], input="".join(f"{a} {s}\n" for a, s in cases), capture_output=True,
                         text=True, check=True).stdout.split()
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
