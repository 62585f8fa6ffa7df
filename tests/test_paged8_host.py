"""Pages of 8 bits without a device: the cache's buffers and the refusals of the operators."""
import pytest
import torch

from dynakv_amd import _lib
from dynakv_amd.kernels.paged import (PagedBatch, PagedKVCache, paged_append, paged_attention,
                                      paged_values)
from dynakv_amd.model import Sampler

CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu
BF = torch.bfloat16


def _batch(max_len=20):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return PagedBatch(i32(0, 1, 2)[None].expand(2, 3).contiguous(), i32(0, 3, 4), i32(20, 5), rows=4,
                      max_new=3, max_len=max_len)


def _codes(pages=4, heads=2, size=16):
    return torch.zeros(pages, heads, size, 128, dtype=torch.uint8).view(CODES)


def _scales(pages=4, heads=2, size=16):
    return torch.zeros(pages, heads, size // 16, dtype=torch.uint8).view(SCALES)


def test_cache_buffers():
    c = PagedKVCache(3, 5, 2, page_size=64, dtype=CODES, device="cpu")
    assert c.k[0].dtype == c.v[2].dtype == CODES and c.k[1].shape == (5, 2, 64, 128)
    assert c.k_scale[0].dtype == c.v_scale[2].dtype == SCALES and len(c.k_scale) == len(c.v_scale) == 3
    assert c.k_scale[1].shape == (5, 2, 4)
    assert len({t.data_ptr() for t in c.k_scale + c.v_scale}) == 6
    assert PagedKVCache(2, 5, 2, device="cpu").k_scale == [None, None]
    with pytest.raises(ValueError, match="unsupported dtype"):
        PagedKVCache(1, 5, 2, dtype=torch.float8_e5m2, device="cpu")


BAD = [dict(k_scale=None), dict(v_scale=None), dict(k_scale=_scales().view(torch.uint8)),
       dict(v_scale=_scales().float()), dict(k_scale=_scales(pages=5)),
       dict(v_scale=_scales(heads=1)), dict(k_scale=_scales(size=32), v_scale=_scales(size=32)),
       dict(k_scale=_scales(heads=4)[:, ::2]), dict(k_pages=_codes().view(torch.uint8)),
       dict(k_pages=torch.zeros(4, 2, 16, 128, dtype=BF), v_pages=torch.zeros(4, 2, 16, 128, dtype=BF)),
       dict(k_scale=None, v_scale=None), dict(v_pages=_codes(heads=1)), dict(batch=_batch(max_len=49))]


@pytest.mark.parametrize("i", range(len(BAD)))
def test_append_and_attention_refusals(i):
    base = dict(k_pages=_codes(), v_pages=_codes(), batch=_batch(), k_scale=_scales(),
                v_scale=_scales())
    q = torch.zeros(4, 4, 128, dtype=BF)
    with pytest.raises(ValueError):
        paged_append(torch.zeros(4, 8 * 128, dtype=BF), heads=4, theta=1e4, **(base | BAD[i]))
    with pytest.raises(ValueError):
        paged_attention(q, **(base | BAD[i]))


def test_other_refusals():
    base = dict(k_pages=_codes(), v_pages=_codes(), batch=_batch(), k_scale=_scales(),
                v_scale=_scales())
    qkv, q = torch.zeros(4, 8 * 128, dtype=BF), torch.zeros(4, 4, 128, dtype=BF)
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged_append(qkv, heads=4, theta=1e4, **base)
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged_attention(q, **base)
    with pytest.raises(ValueError, match="unsupported dtype"):
        paged_append(qkv.float(), heads=4, theta=1e4, **base)
    with pytest.raises(ValueError, match="unsupported dtype"):
        paged_attention(q.to(CODES), **base)
    with pytest.raises(ValueError, match="do not divide"):
        paged_attention(q[:, :3], **base)
    odd = dict(k_pages=_codes(size=24), v_pages=_codes(size=24))
    with pytest.raises(NotImplementedError):
        paged_append(qkv, heads=4, theta=1e4, **(base | odd))
    wide = torch.zeros(4, 2, 64, 4, dtype=torch.uint8).view(SCALES)
    with pytest.raises(ValueError, match="unit last stride"):
        paged_attention(q, **(base | dict(
            k_pages=_codes(size=64), v_pages=_codes(size=64),
            **{n: wide.transpose(2, 3)[:, :, :, 0].view(torch.uint8).as_strided(
                (4, 2, 4), (512, 256, 2)).view(SCALES) for n in ("k_scale", "v_scale")})))


def test_values_refusals():
    base = dict(k_pages=_codes(), v_pages=_codes(), k_scale=_scales(), v_scale=_scales())
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged_values(**base)
    for kw in (dict(k_pages=torch.zeros(4, 2, 16, 128, dtype=BF)), dict(v_pages=_codes(pages=5)),
               dict(k_scale=_scales(pages=5)), dict(dtype=torch.float64), dict(dtype=torch.int32),
               dict(pages=torch.zeros(2, dtype=torch.int64)),
               dict(pages=torch.zeros(2, 2, dtype=torch.int32)),
               dict(pages=torch.zeros(4, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            paged_values(**(base | kw))


def test_c_entry_refusals():
    """The C entries' own checks, which come before anything touches a device."""
    lib = _lib.load()
    E, U, OK, WS = _lib.DKV_E_ARG, _lib.DKV_E_UNSUPPORTED, _lib.DKV_OK, _lib.DKV_E_WORKSPACE
    at = 1 << 32

    def append(dtype=_lib.DKV_BF16, k=at << 1, stride=4096, head=2048, ps=16, ks=at << 2, sp=2, sh=1, B=1,
               T=4, hq=4, hkv=2, q_out=at << 3, norm=at + 2):
        return lib.dkv_paged_append8(None, dtype, at, 1024, q_out, 512, 128, k, k, stride, head, 4, ps,
                                     ks, ks, sp, sh, at << 3, 2, 2, at << 3, at << 3, B, T, hq, hkv,
                                     128, norm, None, 1e-6, at)

    assert append() == U  # (all in order but the norm's weights, off their alignment)
    assert append(ks=None) == E and append(sp=-1) == E and append(sh=0) == E and append(sp=0) == E
    assert append(ps=64, head=8192, stride=16384, sh=3) == E
    assert append(stride=4104) == U and append(head=2056) == U  # (16 bytes)
    assert append(stride=2048, head=1024) == E and append(hq=3) == U and append(dtype=0) == U
    assert append(q_out=at + 16) == E  # on top of the projection
    assert append(B=0) == append(T=0) == OK

    def attend(k=at << 1, stride=4096, ks=at << 2, sp=2, sh=1, q=at, out=at << 3, new=4):
        return lib.dkv_paged_attention8(None, _lib.DKV_BF16, q, 512, 128, k, k, stride, 2048, 4, 16, ks,
                                        ks, sp, sh, at << 3, 4096, 4096, at << 3, at << 3, 1, 4, 4, 2,
                                        128, new, 1, 65536, 0.1, None, 0, out, _lib.DKV_BF16, 512, 128)

    assert attend() == WS and attend(ks=None) == E and attend(sh=0) == E and attend(sp=1 << 40) == WS
    assert attend(stride=4104) == U and attend(k=(at << 1) + 8) == U and attend(out=at + 16) == E
    assert attend(new=0) == OK

    def values(dt=_lib.DKV_BF16, n=4, ids=None, k=at, ks=at << 1, sh=1, ko=at << 2, vo=at << 3, hkv=2):
        return lib.dkv_paged_values(None, dt, k, k, 4096, 2048, 4, 16, hkv, 128, ks, ks, 2, sh, ids, n,
                                    ko, vo)

    assert values(dt=9) == U and values(n=-1) == E and values(n=5) == E and values(hkv=0) == E
    assert values(ks=None) == E and values(sh=0) == E and values(ko=None) == E
    assert values(k=at + 8) == U and values(ko=(at << 2) + 2) == U
    assert values(vo=(at << 2) + 16) == E and values(n=0) == OK  # outputs on top of each other


def test_sampler_penalties_on_the_host():
    s = Sampler(device="cpu")
    assert s.penalties == {} and s._bias is None
    s = Sampler(device="cpu", repetition=1.2, frequency=torch.zeros(2), bias={3: 1.0, 5: -2.0})
    assert set(s.penalties) == {"repetition", "frequency"}
    assert s._bias[0].tolist() == [[3, 5]] and s._bias[1].tolist() == [[1.0, -2.0]]
    s.check(2)
    with pytest.raises(ValueError, match="frequency"):
        s.check(3)
    with pytest.raises(ValueError, match="tokens"):
        s(torch.zeros(2, 10))
