"""``PagedLlama``: the paged append, the attention over the pages and the sampling as one serving loop,
against a float64 forward of the same weights over each request's tokens."""
import math

import pytest
import torch

from dynakv_amd.kernels.sampling import sample_tokens
from dynakv_amd.model import (CompressedLlama, DenseLlama, LlamaShape, PagedLlama, RandomLlama,
                              Sampler)

KW = dict(hidden=512, layers=2, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=1000)


def _logits(model, tokens):
    """(n, vocab) float64 logits after each of the (n,) tokens."""
    s = model.shape
    d = lambda t: t.double()  # noqa: E731
    n, hpg = tokens.shape[0], s.heads // s.kv_heads
    rms = lambda x, w: x / torch.sqrt(x.square().mean(-1, keepdim=True) + s.eps) * d(w)  # noqa: E731
    pos = torch.arange(n, dtype=torch.float64, device=tokens.device)
    freq = torch.tensor([s.theta ** (-2.0 * j / 128) for j in range(64)], dtype=torch.float64,
                        device=tokens.device)
    c, sn = torch.cos(pos[:, None, None] * freq), torch.sin(pos[:, None, None] * freq)

    def turn(x):
        a, b = x[..., :64], x[..., 64:]
        return torch.cat([a * c - b * sn, b * c + a * sn], -1)

    dead = torch.ones(n, n, dtype=torch.bool, device=tokens.device).triu(1)
    x = d(model.embed)[tokens]
    for lw in model.layers:
        h = rms(x, lw.ln1)
        q = (h @ d(lw.wq).T).view(n, s.heads, 128)
        k = (h @ d(lw.wk).T).view(n, s.kv_heads, 128)
        v = (h @ d(lw.wv).T).view(n, s.kv_heads, 128)
        if s.qk_norm:
            q, k = rms(q, lw.q_norm), rms(k, lw.k_norm)
        q, k = turn(q), turn(k)
        a = torch.empty_like(q)
        for i in range(s.heads):
            z = (q[:, i] @ k[:, i // hpg].T / math.sqrt(128)).masked_fill(dead, -math.inf)
            a[:, i] = torch.softmax(z, -1) @ v[:, i // hpg]
        x = x + a.reshape(n, -1) @ d(lw.wo).T
        h = rms(x, lw.ln2)
        x = x + (torch.nn.functional.silu(h @ d(lw.w_gate).T) * (h @ d(lw.w_up).T)) @ d(lw.w_down).T
    return rms(x, model.norm) @ d(model.lm_head).T


def _close(got, want):
    # bf16 weights and activations through two layers: the bound the other models' parity has
    assert float((got.double() - want).abs().max()) <= 0.05 * float(want.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("qk_norm", [False, True])
def test_chunks_beside_tokens_match_the_forward(dev, qk_norm):
    print(f"[gpu] paged model qk_norm={qk_norm}", flush=True)
    m = RandomLlama(LlamaShape(qk_norm=qk_norm, **KW), device=dev, seed=3, std=0.05)
    p = PagedLlama(m, pages=40, page_size=16)
    g = torch.Generator().manual_seed(4)
    tok = lambda n: torch.randint(0, 1000, (n,), generator=g).to(dev)  # noqa: E731
    a, b, c = p.add(), p.add(), p.add()
    seen = {r: torch.empty(0, dtype=torch.long, device=dev) for r in (a, b, c)}

    def step(*feed):
        feed = [(r, tok(n)) for r, n in feed]
        got = p.step(feed)
        for i, (r, t) in enumerate(feed):
            seen[r] = torch.cat([seen[r], t])
            _close(got[i], _logits(m, seen[r])[-1])

    step((a, 70), (b, 5))
    step((a, 1), (b, 60))
    step((c, 33), (a, 1), (b, 1))
    step((a, 1), (b, 1), (c, 1))
    p.end(b)
    step((c, 20), (a, 1))
    assert p.kv_bytes() == 2 * 2 * (5 + 4) * 2 * 16 * 128 * 2  # 73 and 54 tokens in pages of 16
    with pytest.raises(ValueError):
        p.step([])
    with pytest.raises(ValueError):
        p.step([(a, tok(0))])


@pytest.mark.gpu
def test_generate(dev):
    """Greedy tokens are the forward's; a chunk size changes nothing but roundings; the pages come
    back, also from a run that does not fit."""
    print("[gpu] paged generate", flush=True)
    m = RandomLlama(LlamaShape(**KW), device=dev, seed=5, std=0.05)
    p = PagedLlama(m, pages=20, page_size=16)
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 1000, (n,), generator=g).to(dev) for n in (50, 3, 21)]
    for chunk in (512, 16):
        got = p.generate(prompts, 6, chunk=chunk)
        assert got["tokens"].shape == (3, 6) and p.cache.free_pages == 20 and got["pages"] > 0
        for j, t in enumerate(prompts):
            for i in range(6):
                want = _logits(m, torch.cat([t, got["tokens"][j, :i]]))[-1]
                top = float(want.max())
                # within the roundings' reach of the largest
                assert float(want[got["tokens"][j, i]]) >= top - 0.05 * float(want.abs().max())
    with pytest.raises(RuntimeError, match="pages"):
        p.generate([prompts[0].repeat(8)], 2)
    assert p.cache.free_pages == 20
    for bad in (dict(prompts=[], new_tokens=2), dict(prompts=prompts, new_tokens=0),
                dict(prompts=prompts, new_tokens=2, chunk=0),
                dict(prompts=[prompts[0][:0]], new_tokens=2)):
        with pytest.raises(ValueError):
            p.generate(**bad)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["paged", "dense", "compressed"])
def test_generate_with_a_sampler(dev, kind):
    """A seed gives the same tokens again, another one others; a temperature of 0 the largest
    logit's."""
    print(f"[gpu] sampled generate {kind}", flush=True)
    m = RandomLlama(LlamaShape(**KW), device=dev, seed=7, std=0.05)
    g = torch.Generator().manual_seed(8)
    prompt = torch.randint(0, 1000, (2, 30), generator=g).to(dev)
    model = {"paged": lambda: PagedLlama(m, pages=20, page_size=16),
             "dense": lambda: DenseLlama(m, max_len=64), "compressed": lambda: CompressedLlama(m)}
    run = lambda s: model[kind]().generate(  # noqa: E731
        list(prompt) if kind == "paged" else prompt, 8, sampler=s)["tokens"]
    setting = dict(temperature=2.0, top_k=200, top_p=0.95, min_p=0.001)
    first = run(Sampler(seed=1, **setting))
    assert first.shape == (2, 8) and int(first.min()) >= 0 and int(first.max()) < 1000
    assert torch.equal(first, run(Sampler(seed=1, **setting)))
    assert not torch.equal(first, run(Sampler(seed=2, **setting)))
    assert torch.equal(run(Sampler(temperature=0.0)), run(Sampler(top_k=1)))


def test_other_models_refuse_qk_norm():
    class M:
        shape = LlamaShape(qk_norm=True, **KW)

    for kind in (CompressedLlama, DenseLlama):
        with pytest.raises(ValueError, match="query and key norms"):
            kind(M())


@pytest.mark.gpu
def test_a_sampler_gives_tokens_that_can_be_looked_up(dev):
    """A row of NaN or -infinity has no token (-1): the generators' sampler gives token 0 for it."""
    print("[gpu] sampler without tokens", flush=True)
    logits = torch.randn(4, 50, device=dev)
    logits[1], logits[2] = float("nan"), float("-inf")
    assert sample_tokens(logits, torch.full((4,), 0.5, device=dev)).tolist()[1:3] == [-1, -1]
    t = Sampler(seed=3, device=dev)(logits)
    assert t[1:3].tolist() == [0, 0] and int(t.min()) >= 0


@pytest.mark.gpu
def test_generate_with_settings_of_each_request(dev, monkeypatch):
    """Settings with an entry per request hold for that request in every step, whichever others are in
    it, and its uniform numbers are its own: the same for every size of chunk."""
    print("[gpu] sampled generate, settings of each request", flush=True)
    m = RandomLlama(LlamaShape(**KW), device=dev, seed=9, std=0.05)
    p = PagedLlama(m, pages=20, page_size=16)
    g = torch.Generator().manual_seed(10)
    prompts = [torch.randint(0, 1000, (n,), generator=g).to(dev) for n in (50, 3, 21, 40)]
    f32 = lambda *v: torch.tensor(v, dtype=torch.float32, device=dev)  # noqa: E731
    setting = dict(temperature=f32(0.0, 50.0, 1.0, 1.0), top_p=f32(1.0, 1.0, 1.0, 0.0),
                   top_k=torch.tensor([0, 0, 1, 0], dtype=torch.int32, device=dev))
    for chunk in (512, 16):
        got = p.generate(prompts, 5, Sampler(seed=3, **setting), chunk=chunk)["tokens"]
        assert got.shape == (4, 5) and p.cache.free_pages == 20
        near = []
        for j, t in enumerate(prompts):
            want = [_logits(m, torch.cat([t, got[j, :i]]))[-1] for i in range(5)]
            near.append([float(w[got[j, i]]) >= float(w.max()) - 0.05 * float(w.abs().max())
                         for i, w in enumerate(want)])
        # greedy by temperature, by top-k, by top-p; and one that is nearly uniform over 1000 tokens
        assert all(near[0]) and all(near[2]) and all(near[3]) and not all(near[1])
    # tokens that the uniform numbers alone decide
    seen = []

    def by_u(logits, u, **kw):
        seen.append((logits.shape[0], {k: v.tolist() for k, v in kw.items() if torch.is_tensor(v)}))
        return (u * 1000).long()

    monkeypatch.setattr("dynakv_amd.model.sample_tokens", by_u)
    runs = [p.generate(prompts, 5, Sampler(seed=4, **setting), chunk=c)["tokens"]
            for c in (512, 16, 1, 512)]
    for r in runs[1:]:
        assert torch.equal(r, runs[0])
    assert len(set(runs[0].flatten().tolist())) > 15
    top_p = setting["top_p"].tolist()
    for rows, kw in seen:
        assert rows > 0 and all(len(v) == rows for v in kw.values())
    assert seen[0][1]["top_p"] == top_p
    # one entry too few: refused before anything is fed
    with pytest.raises(ValueError, match="entry"):
        p.generate(prompts[:3], 5, Sampler(seed=3, **setting))
    assert p.cache.free_pages == 20
    # as a callable of its own: rows of some requests
    logits = torch.randn(2, 1000, device=dev)
    monkeypatch.undo()
    s = Sampler(seed=3, **setting)
    assert torch.equal(s(logits, requests=[2, 0]), logits.argmax(-1))
    with pytest.raises(ValueError):
        s(logits, requests=[2, 4])
    with pytest.raises(ValueError):
        s(logits, requests=[0, -1])
    with pytest.raises(ValueError):
        s(logits, requests=[0])
