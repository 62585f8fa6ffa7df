"""Pages read back over the whole range of codes and scales: what is not a number of the result's type is
rounded to its nearest one (half of the largest step past the largest and on: infinity)."""
import pytest
import torch

from dynakv_amd.kernels.paged import paged_values

CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_values_of_every_code_and_scale(dev, dtype):
    """All 256 codes under all 256 scales. Their products have four bits, so that fp32 holds all that is not
    past its largest number, and one rounding from there is the nearest value."""
    print(f"[gpu] paged values of every code {dtype}", flush=True)
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8).repeat(16 * 16, 8)  # block: every code 8x
    codes = codes.view(16, 1, 256, 128).to(dev)
    byte = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(16, 1, 16).to(dev)
    k, v = paged_values(codes.view(CODES), codes.flip(-1).contiguous().view(CODES), byte.view(SCALES),
                        byte.view(SCALES), dtype=dtype)
    for got, c in ((k, codes), (v, codes.flip(-1))):
        two = torch.ldexp(torch.ones(256, dtype=torch.float64), torch.arange(256) - 127)
        two[255] = float("nan")
        exact = c.cpu().view(CODES).double() * two.view(16, 1, 16).repeat_interleave(16, -1)[..., None]
        want, got = exact.float().to(dtype), got.cpu()
        same = (got == want) | (got.isnan() & want.isnan())
        wrong = sorted({(int(b), float(x), float(y)) for b, x, y in zip(
            byte.cpu().view(16, 1, 16).repeat_interleave(16, -1)[..., None].expand(same.shape)[~same],
            want[~same], got[~same])})
        print(f"[gpu]   {len(wrong)} wrong, scales {sorted({w[0] for w in wrong})} {wrong[:3]} {wrong[-3:]}",
              flush=True)
        assert bool(same.all())
