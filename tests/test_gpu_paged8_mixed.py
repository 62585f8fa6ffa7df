"""Pages whose scales lie outside the range of the type that is appended to them (those of a model in another
type, or a user's own): the earlier tokens keep their values as far as the range holds them."""
import math

import pytest
import torch

from dynakv_amd.kernels.paged import paged_append, paged_values
from test_gpu_paged8 import BF, CODES, DH, FP, RANGE, Step8, nearest, two_to, u8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("first", [1, 9, 15])
def test_append_to_blocks_of_any_scale(dev, dtype, first):
    """Blocks with ``first`` earlier tokens of every code, under all 256 scales. Below the range, or where the new
    token asks for more, codes are rounded again to the new scale; above it, to the largest of the range, at most
    448 times it; a NaN scale's tokens are NaN."""
    print(f"[gpu] paged append8 any scale {dtype} {first}", flush=True)
    low, high = RANGE[dtype]
    for size in (2.0**-10, 1.0):
        s = Step8(dev, [1] * 256, [first + 1] * 256, hkv=2, dtype=dtype, seed=81, data=False)
        pages = s.table[:, 0].long().to(dev)
        byte = torch.arange(256, dtype=torch.int32).to(torch.uint8).to(dev)
        g = torch.Generator().manual_seed(8)
        for codes, scale in ((s.k, s.k_scale), (s.v, s.v_scale)):
            c = torch.randint(0, 256, (256, 2, first, DH), generator=g, dtype=torch.uint8).to(dev)
            codes.view(torch.uint8)[pages, :, :first] = c
            scale.view(torch.uint8)[pages] = byte[:, None, None]
        before = {n: u8(t)[pages].clone() for n, t in (("k", s.k), ("v", s.v))}
        qkv = (s.rand(256, 4 * 2 * DH).float() * size).to(dtype)
        paged_append(qkv, s.k, s.v, s.batch, heads=4, theta=1e4, **s.both)
        held = paged_values(s.k, s.v, **s.both, pages=pages.int(), dtype=torch.float32)
        for name, scale, now in (("k", s.k_scale, held[0]), ("v", s.v_scale, held[1])):
            e = u8(scale)[pages][..., 0].long() - 127                      # (256, 2)
            old = torch.arange(256, device=dev)[:, None].expand(256, 2) - 127
            big = now[:, :, first].double().abs().amax(-1)  # (held: at least half the new token's largest)
            assert bool(((e >= low) & (e <= high) & (e >= old.clamp(low, high))).all())
            least = (e == old.clamp(low, high)) | (2.0 * big > two_to(e) * 224)
            assert bool((least | (old == 128)).all())
            was = before[name][:, :, :first].contiguous().view(CODES).double()
            x = was * two_to((old - e).clamp(-1000, 1000))[..., None, None]
            want = nearest(x.nan_to_num()) * two_to(e)[..., None, None]
            want = torch.where(was.isnan() | (old == 128)[..., None, None], math.nan, want)
            got = now[:, :, :first].double()
            same = (got == want) | (got.isnan() & want.isnan())
            wrong = torch.nonzero(~same)[:, 0].unique().tolist()
            assert not wrong, (name, wrong[:5], wrong[-5:])
            assert torch.equal(u8(getattr(s, name))[pages][:, :, first + 1:], before[name][:, :, first + 1:])
            # scales that stay leave the codes as they are, to the bit
            kept = (e == old)[..., None, None]
            codes = u8(getattr(s, name))[pages][:, :, :first]
            assert bool(((codes == before[name][:, :, :first]) | ~kept).all())
