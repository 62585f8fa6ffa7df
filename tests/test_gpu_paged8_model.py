"""``PagedLlama`` over 8-bit pages, and samplers with penalties in the generators."""
import math

import pytest
import torch

from dynakv_amd.model import (CompressedLlama, DenseLlama, LlamaShape, PagedLlama, RandomLlama,
                              Sampler)
from test_gpu_paged8 import CODES, nearest, two_to

KW = dict(hidden=512, layers=2, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=1000)


def _held(x):
    """(n, heads, 128) float64 as blocks of 16 tokens of a head hold them."""
    out = torch.empty_like(x)
    for t0 in range(0, x.shape[0], 16):
        b = x[t0:t0 + 16]
        m, e = torch.frexp(b.abs().amax((0, 2)) / 448)
        two = two_to(e - (m == 0.5).int())[None, :, None]
        out[t0:t0 + 16] = nearest(b / two) * two
    return out


class _Oracle:
    """The two operators in float64, on the activations that the model has: requests' keys and values kept
    aside by their first page, held as blocks of 16 when they are attended."""

    def __init__(self):
        self.kept = {}

    def _requests(self, batch):
        starts, lens = batch.q_start.tolist(), batch.lens.tolist()
        for b, (i, j, n) in enumerate(zip(starts, starts[1:], lens)):
            yield int(batch.page_table[b, 0]), i, j, n

    def append(self, qkv, k_pages, v_pages, batch, *, heads, theta, q_norm, k_norm, eps, k_scale,
               v_scale):
        hkv = k_pages.shape[1]
        x = qkv.double().view(qkv.shape[0], -1, 128)
        freq = torch.tensor([theta ** (-2.0 * j / 128) for j in range(64)], dtype=torch.float64,
                            device=x.device)
        q = torch.empty_like(x[:, :heads])
        for who, i, j, n in self._requests(batch):
            ang = torch.arange(n - j + i, n, dtype=torch.float64, device=x.device)[:, None, None] * freq
            y, c, sn = x[i:j, :heads + hkv], torch.cos(ang), torch.sin(ang)
            y = torch.cat([y[..., :64] * c - y[..., 64:] * sn, y[..., 64:] * c + y[..., :64] * sn], -1)
            q[i:j] = y[:, :heads]
            new = torch.stack([y[:, heads:], x[i:j, heads + hkv:]])
            old = self.kept.get((id(k_pages), who))
            if old is not None and n > j - i:
                new = torch.cat([old[:, :n - j + i], new], 1)
            self.kept[id(k_pages), who] = new
        return q.to(qkv.dtype)

    def attention(self, q, k_pages, v_pages, batch, *, k_scale, v_scale):
        out = torch.empty_like(q)
        hpg = q.shape[1] // k_pages.shape[1]
        for who, i, j, n in self._requests(batch):
            k, v = (_held(t).repeat_interleave(hpg, 1).transpose(0, 1)
                    for t in self.kept[id(k_pages), who])
            z = torch.matmul(q[i:j].double().transpose(0, 1), k.transpose(1, 2).contiguous())
            pos = torch.arange(n, device=q.device)
            z = (z / math.sqrt(128)).masked_fill(pos[None] > pos[n - j + i:, None], -math.inf)
            out[i:j] = torch.matmul(torch.softmax(z, -1), v).transpose(0, 1).to(q.dtype)
        return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_chunks_beside_tokens_match_the_formulas(dev, dtype, monkeypatch):
    """A step against the same model over the formulas in float64 (over a forward in float64 it would not
    do: 16-bit activations put one key in twenty on the other side of a border between two codes, a step of
    2^-3). The operators' results differ by at most a rounding of their 16-bit output, a small part of
    what the bound of the 16-bit cache's test (roundings through two layers) allows."""
    print(f"[gpu] paged8 model {dtype}", flush=True)
    m = RandomLlama(LlamaShape(**KW), device=dev, seed=3, std=0.05, dtype=dtype)
    p, ref = (PagedLlama(m, pages=40, page_size=16, cache_dtype=CODES) for _ in range(2))
    assert p.cache.k[0].dtype == CODES
    oracle = _Oracle()
    g = torch.Generator().manual_seed(4)
    tok = lambda n: torch.randint(0, 1000, (n,), generator=g).to(dev)  # noqa: E731
    (a, b, c), ids = ([x.add() for _ in range(3)] for x in (p, ref))
    same = dict(zip((a, b, c), ids))

    def step(*feed):
        feed = [(r, tok(n)) for r, n in feed]
        got = p.step(feed)
        with monkeypatch.context() as patch:
            patch.setattr("dynakv_amd.model.paged_append", oracle.append)
            patch.setattr("dynakv_amd.model.paged_attention", oracle.attention)
            want = ref.step([(same[r], t) for r, t in feed]).double()
        fine = (got.double() - want).abs().amax(-1) <= 0.05 * want.abs().amax(-1)
        assert bool(fine.all())

    step((a, 70), (b, 5))
    step((a, 1), (b, 60))
    step((c, 33), (a, 1), (b, 1))
    step((a, 1), (b, 1), (c, 1))
    p.end(b), ref.end(same[b])
    step((c, 20), (a, 1))
    # 73 and 54 tokens in pages of 16: a byte a value and one for each 16 tokens
    assert p.kv_bytes() == 2 * 2 * (5 + 4) * 2 * 16 * 128 + 2 * 2 * (5 + 4) * 2


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["paged", "paged8", "dense", "compressed"])
def test_generate_with_penalties(dev, kind):
    """With a presence penalty that outweighs everything no token comes twice; with a repetition penalty
    none of the prompt's either; a bias alone decides; settings of each request are the request's."""
    print(f"[gpu] penalties {kind}", flush=True)
    m = RandomLlama(LlamaShape(**KW), device=dev, seed=7, std=0.05)
    g = torch.Generator().manual_seed(8)
    prompt = torch.randint(0, 1000, (2, 30), generator=g).to(dev)
    model = {"paged": lambda: PagedLlama(m, pages=20, page_size=16),
             "paged8": lambda: PagedLlama(m, pages=20, page_size=16, cache_dtype=CODES),
             "dense": lambda: DenseLlama(m, max_len=80), "compressed": lambda: CompressedLlama(m)}
    run = lambda **kw: model[kind]().generate(  # noqa: E731
        list(prompt) if kind.startswith("paged") else prompt, 12,
        sampler=Sampler(temperature=0.0, **kw))["tokens"]
    got = run(presence=1e4)
    for row in got:
        assert len(set(row.tolist())) == 12
    got = run(repetition=1e4, presence=1e4)
    for row, p in zip(got, prompt):
        assert len(set(row.tolist())) == 12 and not set(row.tolist()) & set(p.tolist())
    assert bool((run(bias={7: 1e4}) == 7).all())
    f32 = lambda *v: torch.tensor(v, dtype=torch.float32, device=dev)  # noqa: E731
    got = run(bias={7: 1e4, 9: 9e3}, presence=f32(0.0, 5e3), frequency=f32(0.0, 1.0))
    assert bool((got[0] == 7).all())
    assert got[1, :3].tolist() == [7, 9, 7]  # 1e4, then 9e3 against 1e4 - 5e3 - 1, then 4999 to 3999
    with pytest.raises(ValueError, match="tokens"):
        Sampler(presence=1.0)(torch.zeros(2, 1000, device=dev))
    allowed = torch.zeros(2, 32, dtype=torch.int32, device=dev)
    allowed[0, 3], allowed[1, 0] = 1 << 5, 2
    logits = torch.randn(2, 1, 1000, device=dev)
    before = logits.clone()
    assert Sampler()(logits, allowed=allowed).tolist() == [[101], [1]]
    assert torch.equal(logits, before)


@pytest.mark.gpu
def test_generate_of_different_lengths_with_penalties(dev):
    """Prompts of different lengths, in chunks: a request's penalties are over its own tokens."""
    print("[gpu] penalties ragged", flush=True)
    m = RandomLlama(LlamaShape(**KW), device=dev, seed=9, std=0.05)
    g = torch.Generator().manual_seed(10)
    prompts = [torch.randint(0, 1000, (n,), generator=g).to(dev) for n in (50, 3, 21)]
    make = lambda: Sampler(temperature=0.0, repetition=1.3, frequency=0.2, presence=0.1)  # noqa: E731
    together = PagedLlama(m, pages=30, page_size=16).generate(prompts, 10, make(), chunk=16)["tokens"]
    for j, p in enumerate(prompts):
        alone = PagedLlama(m, pages=30, page_size=16)
        r, out, feed = alone.add(), [], p
        for i in range(10):
            logits = alone.step([(r, feed)])
            tokens = torch.cat([p, torch.tensor(out, dtype=torch.long, device=dev)])[None]
            tok = make()(logits, tokens=tokens, prompt_lens=p.shape[0], lens=p.shape[0] + i)
            # another batch rounds the logits otherwise: compared while the tokens agree so far
            if int(tok) != int(together[j, i]):
                top = logits[0].float().topk(2).values
                assert float(top[0] - top[1]) < 0.5, (j, i)
                break
            out.append(int(tok))
            feed = tok
