"""Which launches and which workspace the attention takes of 8-bit pages, and that 16-bit pages keep theirs."""
import pytest
import torch

from dynakv_amd import _lib
from dynakv_amd.kernels import paged
from dynakv_amd.kernels.paged import PagedBatch, paged_attention

CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.mark.parametrize("B", [1, 31, 32, 40, 63, 64, 300])
def test_workspace_by_the_kind_of_pages(B):
    """32 to 63 requests of 8 KV heads are cut where their pages are of 8 bits, and only there: of 16 bits a
    unit is one workgroup's, without records."""
    lib = _lib.load()
    of = lambda bits: lib.dkv_paged_workspace_floats_of(bits, B, B, 32, 8, 1, 1, 8192)  # noqa: E731
    assert (of(16) > 0) == (B < 32) and (of(8) > 0) == (B < 64)
    assert lib.dkv_paged_workspace_floats(B, B, 32, 8, 1, 1, 8192) == max(of(8), of(16))
    assert lib.dkv_paged_workspace_floats_of(16, B, B, 32, 7, 1, 1, 8192) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("module", [True, False])
def test_a_call_without_records_takes_no_workspace(dev, monkeypatch, module):
    print(f"[gpu] paged workspace of 40 requests, tensor module {module}", flush=True)
    if not module:
        monkeypatch.setattr(_lib, "_tensor_calls", None)
    asked, inner = [], paged._attention_workspace
    monkeypatch.setattr(paged, "_attention_workspace", lambda *a: asked.append(a[2]) or inner(*a))
    B, i32 = 40, lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    # (from 512 tokens on: 16 tiles, the least part)
    batch = PagedBatch(i32([list(range(63))] * B), i32(list(range(B + 1))), i32([1000] * B), rows=B,
                       max_new=1, max_len=1000)
    q = torch.randn(B, 32, 128, device=dev).bfloat16()
    k = torch.zeros(63, 8, 16, 128, dtype=torch.bfloat16, device=dev)
    paged_attention(q, k, k.clone(), batch)
    assert asked == []
    scale = torch.full((63, 8, 1), 127, dtype=torch.uint8, device=dev).view(SCALES)
    paged_attention(q, k.to(CODES), k.to(CODES), batch, k_scale=scale, v_scale=scale.clone())
    assert len(asked) == 1 and asked[0] > 0
