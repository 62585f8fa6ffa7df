"""Performance cases of the serving operators: a paged cache, the attention that reads it, sampling.

A serving step takes the requests at hand, each with new tokens of its own number (a chunk of its
prompt, or the one token it generated), through three operators: ``append`` norms (where the model
has such norms) and rotates the step's queries and keys and writes keys and values to the
requests' pages, ``attend`` lets the new tokens attend their requests' pages, and ``sample`` draws
each request's next token from its logits.

``listed`` has the fixed cases, ``draw`` further ones of the same ranges. ``prepare`` builds a
case's inputs from a seed, ``run`` is one pass (plain torch, or the package's operators where
``own`` is set), ``work`` the bytes and operations a pass cannot do without, ``exact`` the same
outputs in float64.
"""

from __future__ import annotations

import math

import torch

own = False

DH = 128            # head dimension
THETA = 500000.0
EPS = 1e-6          # of the query and key norms
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one decode step of 16 users at up to 8K tokens
        dict(name="append_step", op="append", dtype="bf16", groups=8, heads=32, page=64,
             requests=16, new=1, most=8192, ragged=True, norms=False),
        # the first chunk of a user's prompt far into a document, with query and key norms
        dict(name="append_chunk", op="append", dtype="fp16", groups=4, heads=16, page=16,
             requests=1, new=777, most=100001, ragged=False, norms=True),
        # four 2048-token prompts
        dict(name="append_prompt", op="append", dtype="bf16", groups=8, heads=32, page=64,
             requests=4, new=2048, most=2048, ragged=False, norms=True),
        # the first tokens of one user's chat: a launch whose latency is all there is
        dict(name="attend_tiny", op="attend", dtype="bf16", groups=8, heads=32, page=16,
             requests=1, new=1, most=96, ragged=False, chunks=0),
        # the benchmark's batch: 16 users decoding over up to 8K tokens each
        dict(name="attend_step", op="attend", dtype="bf16", groups=8, heads=32, page=64,
             requests=16, new=1, most=8192, ragged=True, chunks=0),
        # two users decoding over long documents, odd lengths
        dict(name="attend_long", op="attend", dtype="fp16", groups=8, heads=32, page=128,
             requests=2, new=1, most=65533, ragged=False, chunks=0),
        # prefill of four 2048-token prompts
        dict(name="attend_prompt", op="attend", dtype="bf16", groups=8, heads=32, page=64,
             requests=4, new=2048, most=2048, ragged=False, chunks=0),
        # the later chunks of two long prompts, 16-token pages
        dict(name="attend_chunk", op="attend", dtype="fp16", groups=8, heads=32, page=16,
             requests=2, new=500, most=6001, ragged=True, chunks=0),
        # users decoding while one user's prompt goes through in a chunk
        dict(name="attend_mixed", op="attend", dtype="bf16", groups=4, heads=16, page=32,
             requests=12, new=1, most=4096, ragged=True, chunks=512),
        # one user's next token under the usual filters
        dict(name="sample_one", op="sample", dtype="bf16", rows=1, vocab=32000, filters="all"),
        # a batch of users, each with settings of its own, fp32 logits
        dict(name="sample_mixed", op="sample", dtype="fp32", rows=37, vocab=50257,
             filters="mixed"),
        # a large batch over a large vocabulary, nucleus sampling
        dict(name="sample_batch", op="sample", dtype="bf16", rows=256, vocab=128256,
             filters="top_p"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["append", "attend", "attend", "attend", "sample"])
    if op == "sample":
        return dict(op="sample", dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    rows=_log_int(rng, 1, 128), vocab=_log_int(rng, 1000, 128256),
                    filters=rng.choice(["all", "mixed", "top_p", "top_k", "min_p", "none",
                                        "greedy"]))
    groups, heads = rng.choice([(8, 32), (8, 32), (4, 16), (2, 4), (8, 8), (2, 14)])
    base = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), groups=groups, heads=heads,
                page=rng.choice([16, 32, 64, 128]))
    kind = rng.choice(["step", "few", "prompt", "chunk", "mixed"])
    if op == "append":
        # a step's tokens to a batch of prompts, near and far positions
        if kind in ("step", "few", "mixed"):
            return base | dict(requests=_log_int(rng, 1, 64), new=1 if kind == "step" else
                               rng.randint(2, 9), most=_log_int(rng, 64, 8192), ragged=True,
                               norms=rng.random() < 0.5)
        new = _log_int(rng, 33, 2048)
        return base | dict(requests=rng.randint(1, 3), new=new,
                           most=new if kind == "prompt" else new + _log_int(rng, 1, 30000),
                           ragged=rng.random() < 0.5, norms=rng.random() < 0.5)
    if kind in ("step", "few"):
        # single tokens, or a few drafted ones, of one to 16 users over short and long caches
        requests = _log_int(rng, 1, 16)
        new = 1 if kind == "step" else rng.randint(2, 9)
        most = _log_int(rng, 17, 8000 if requests > 2 else 32768)
        return base | dict(requests=requests, new=min(new, most), most=most,
                           ragged=rng.random() < 0.7, chunks=0)
    if kind == "mixed":
        return base | dict(requests=rng.randint(2, 12), new=1, most=_log_int(rng, 600, 4096),
                           ragged=True, chunks=_log_int(rng, 33, 512))
    new = _log_int(rng, 33, 1000)
    return base | dict(requests=rng.randint(1, 2), new=new,
                       most=new if kind == "prompt" else new + _log_int(rng, 1, 3500),
                       ragged=rng.random() < 0.5, chunks=0)


def _lens(case) -> tuple[list[int], list[int]]:
    """(new tokens, tokens with them) of each request, by the case alone: a ragged batch's caches
    hold between a quarter of ``most`` and all of it, its chunks between half of ``new`` and all."""
    new, lens = [], []
    n = case["requests"]
    for b in range(n):
        part = ((b * 0.6180339887) % 1.0) if case["ragged"] and n > 1 else 0.0
        new.append(max(1, round(case["new"] * (1.0 - 0.5 * part))))
        cached = case["most"] - case["new"]
        lens.append(new[b] + round(cached * (1.0 - 0.75 * part)))
    if case.get("chunks"):  # one more request, in the middle, with a chunk of its prompt
        new.insert(n // 2, case["chunks"])
        lens.insert(n // 2, max(case["chunks"], case["most"] // 2))
    return new, lens


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(1_000_003 * (int(seed) + 1))
    return g


def _normal(g, *dims, dtype) -> torch.Tensor:
    return torch.randn(*dims, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _ints(v) -> torch.Tensor:
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def _batch(case, g) -> dict:
    """The step's plan: page table over pages in the order a pool hands them out after some use
    (any order), row ranges, lengths."""
    new, lens = _lens(case)
    page = case["page"]
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    ids = torch.randperm(total, generator=g, device=DEV)
    table = torch.full((len(new), max(need)), -1, device=DEV, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n].to(torch.int32)
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return dict(table=table, q_start=_ints(starts), lens=_ints(lens), rows=starts[-1],
                max_new=max(new), min_new=min(new), max_len=max(lens), pages=total)


def _pool(case, g, pages: int) -> tuple[torch.Tensor, torch.Tensor]:
    dims = (pages, case["groups"], case["page"], DH)
    dt = DTYPES[case["dtype"]]
    return _normal(g, *dims, dtype=dt), _normal(g, *dims, dtype=dt)


def _sample_inputs(case, g) -> dict:
    rows, vocab = case["rows"], case["vocab"]
    # a language model's logits: a broad body, and a few tokens far above it, more so in some rows
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 2.5
    top = torch.randint(0, vocab, (rows, 40), generator=g, device=DEV)
    lift = 6.0 + 4.0 * torch.rand(rows, 1, generator=g, device=DEV)
    x.scatter_add_(1, top, lift * torch.rand(rows, 40, generator=g, device=DEV))
    r = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device=DEV)  # noqa: E731
    u = torch.rand(rows, generator=g, device=DEV)
    temperature = r(0.6, 1.2)
    top_k = torch.randint(20, 200, (rows,), generator=g, device=DEV, dtype=torch.int32)
    top_p, min_p = r(0.7, 0.99), r(0.01, 0.1)
    f = case["filters"]
    if f == "mixed":  # each row leaves filters out at random; every fifth is greedy
        pick = torch.rand(4, rows, generator=g, device=DEV)
        top_k[pick[0] < 0.5] = 0
        top_p[pick[1] < 0.5] = 1.0
        min_p[pick[2] < 0.5] = 0.0
        temperature[pick[3] < 0.2] = 0.0
    if f in ("top_p", "min_p", "none", "greedy"):
        top_k.zero_()
    if f in ("top_k", "min_p", "none", "greedy"):
        top_p.fill_(1.0)
    if f in ("top_k", "top_p", "none", "greedy"):
        min_p.zero_()
    if f == "greedy":
        temperature.zero_()
    return dict(logits=x.to(DTYPES[case["dtype"]]), u=u, temperature=temperature, top_k=top_k,
                top_p=top_p, min_p=min_p)


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "sample":
        return dict(case=case) | _sample_inputs(case, g)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case) | _batch(case, g)
    s["k"], s["v"] = _pool(case, g, s["pages"])
    if case["op"] == "attend":
        s["q"] = _normal(g, s["rows"], case["heads"], DH, dtype=dt)
        return s
    s["qkv"] = _normal(g, s["rows"], (case["heads"] + 2 * case["groups"]) * DH, dtype=dt)
    s["q_norm"] = s["k_norm"] = None
    if case["norms"]:
        s["q_norm"] = (1.0 + 0.1 * torch.randn(DH, generator=g, device=DEV)).to(dt)
        s["k_norm"] = (1.0 + 0.1 * torch.randn(DH, generator=g, device=DEV)).to(dt)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[op](state)


def _run_own(s):
    case = s["case"]
    if case["op"] == "sample":
        from dynakv_amd.kernels.sampling import sample_tokens
        return sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                             top_p=s["top_p"], min_p=s["min_p"])
    from dynakv_amd.kernels.paged import PagedBatch, paged_append, paged_attention
    batch = PagedBatch(page_table=s["table"], q_start=s["q_start"], lens=s["lens"],
                       rows=s["rows"], max_new=s["max_new"], max_len=s["max_len"],
                       min_new=s["min_new"])
    if case["op"] == "attend":
        return paged_attention(s["q"], s["k"], s["v"], batch)
    q = paged_append(s["qkv"], s["k"], s["v"], batch, heads=case["heads"], theta=THETA,
                     q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    return dict(q=q, k=s["k"], v=s["v"])


def _places(s):
    """(request, position) of each row of the step."""
    row = torch.arange(s["rows"], device=DEV)
    req = torch.bucketize(row, s["q_start"][1:].long(), right=True)
    return req, s["lens"][req].long() - s["q_start"][req + 1].long() + row


def _plain_append(s):
    case = s["case"]
    hq, g, page = case["heads"], case["groups"], case["page"]
    req, pos = _places(s)
    x = s["qkv"].float().view(s["rows"], hq + 2 * g, DH)
    q, k, v = x[:, :hq], x[:, hq:hq + g], s["qkv"].view(s["rows"], hq + 2 * g, DH)[:, hq + g:]
    if s["q_norm"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"].float()
    j = torch.arange(DH // 2, device=DEV, dtype=torch.float64)
    # far positions times frequencies: the angle in 64 bits
    ang = pos.double()[:, None] * torch.exp(-(2.0 * j / DH) * math.log(THETA))
    c, sn = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]

    def turn(t):
        a, b = t[..., : DH // 2], t[..., DH // 2:]
        return torch.cat([a * c - b * sn, b * c + a * sn], dim=-1).to(s["qkv"].dtype)

    where = s["table"][req, pos // page].long()[:, None]
    slot, head = (pos % page)[:, None], torch.arange(g, device=DEV)[None, :]
    s["k"][where, head, slot] = turn(k)
    s["v"][where, head, slot] = v
    return dict(q=turn(q), k=s["k"], v=s["v"])


def _plain_attend(s):
    case = s["case"]
    hq, g, page = case["heads"], case["groups"], case["page"]
    hpg, n_max, l_max = hq // g, s["max_new"], s["max_len"]
    req, pos = _places(s)
    key = torch.arange(l_max, device=DEV)
    where = s["table"][:, key // page].long()                      # (B, L); -1 past the request
    inside = key < s["lens"][:, None]                              # (B, L)
    pick = lambda t: torch.where(inside[:, :, None, None], t[where, :, key % page].float(),  # noqa: E731
                                 0.0).transpose(1, 2)              # (B, G, L, DH)
    k, v = pick(s["k"]), pick(s["v"])
    # rows of the step as (B, G, new token and head of the group, DH), padded to the longest
    at = torch.arange(s["rows"], device=DEV) - s["q_start"][req].long()
    n = s["lens"].numel()
    q = torch.zeros(n, n_max, hq, DH, device=DEV)
    q[req, at] = s["q"].float()
    limit = torch.full((n, n_max), -1, device=DEV)
    limit[req, at] = pos
    q = q.view(n, n_max, g, hpg, DH).transpose(1, 2).reshape(n, g, n_max * hpg, DH)
    dead = key > limit.repeat_interleave(hpg, 1)[:, None, :, None]  # (B, 1, rows, L)
    z = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(DH))
    z.masked_fill_(dead, -math.inf)
    m = z.amax(-1, keepdim=True)
    e = z.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    o = o.view(n, g, n_max, hpg, DH).transpose(1, 2).reshape(n, n_max, hq, DH)
    return o[req, at].to(s["q"].dtype)


def _plain_sample(s):
    x = s["logits"].double()
    # largest first, of equal ones the lowest index first
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    best = order.indices[:, 0]
    t = s["temperature"].double()[:, None]
    greedy = t == 0
    w = torch.exp((order.values - order.values[:, :1]) / torch.where(greedy, 1.0, t))
    rank = torch.arange(x.shape[1], device=DEV)[None, :]
    k = s["top_k"].long()[:, None]
    w = torch.where((rank < k) | (k <= 0), w, 0.0)
    before = torch.cumsum(w, -1) - w
    p = s["top_p"].double()[:, None]
    keep = (before < p * w.sum(-1, keepdim=True)) | (p >= 1) | (rank == 0)
    keep &= (w >= s["min_p"].double()[:, None]) | (rank == 0)
    w = torch.where(keep, w, 0.0)
    # the running mass in the vocabulary's own order
    mass = torch.zeros_like(x).scatter_(1, order.indices, w)
    run_ = torch.cumsum(mass, -1)
    hit = run_ > s["u"].double()[:, None] * run_[:, -1:]
    return torch.where(greedy[:, 0], best, (~hit).sum(-1))


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case) -> dict:
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["rows"] * case["vocab"]
        return dict(bytes=size * n + 28 * case["rows"], flops=4 * n)
    new, lens = _lens(case)
    rows, hq, g = sum(new), case["heads"], case["groups"]
    if case["op"] == "append":
        vals = rows * (hq + 2 * g) * DH
        return dict(bytes=2 * 2 * vals, flops=(8 if case["norms"] else 4) * vals)
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, lens))
    return dict(bytes=2 * (2 * sum(lens) * g * DH + 2 * rows * hq * DH),
                flops=4 * pairs * hq * DH)


# ---------------------------------------------------------------------------------------------
# float64 results
# ---------------------------------------------------------------------------------------------
def _exact_append(s, case):
    hq, g, page = case["heads"], case["groups"], case["page"]
    new, lens = _lens(case)
    table = s["table"].tolist()
    kp, vp = s["k"].double(), s["v"].double()
    q_out = torch.empty(s["rows"], hq, DH, device=DEV, dtype=torch.float64)
    freq = torch.tensor([THETA ** (-2.0 * i / DH) for i in range(DH // 2)], device=DEV,
                        dtype=torch.float64)
    at = 0
    for b, (n, total) in enumerate(zip(new, lens)):
        x = s["qkv"][at:at + n].double().view(n, hq + 2 * g, DH)
        y = x[:, :hq + g].clone()
        if s["q_norm"] is not None:
            y /= torch.sqrt((y * y).sum(-1, keepdim=True) / DH + EPS)
            y[:, :hq] *= s["q_norm"].double()
            y[:, hq:] *= s["k_norm"].double()
        ang = torch.arange(total - n, total, device=DEV, dtype=torch.float64)[:, None, None] * freq
        # a pair (j, j + 64) as a complex number, turned by its angle
        z = torch.complex(y[..., : DH // 2], y[..., DH // 2:]) * torch.polar(
            torch.ones_like(ang), ang)
        y = torch.cat([z.real, z.imag], dim=-1)
        q_out[at:at + n] = y[:, :hq]
        for p0 in range((total - n) // page * page, total, page):  # page by page
            lo, hi = max(p0, total - n), min(p0 + page, total)
            rows = slice(lo - (total - n), hi - (total - n))
            kp[table[b][p0 // page], :, lo - p0:hi - p0] = y[rows, hq:].transpose(0, 1)
            vp[table[b][p0 // page], :, lo - p0:hi - p0] = x[rows, hq + g:].transpose(0, 1)
        at += n
    return dict(q=q_out, k=kp, v=vp)


def _exact_attend(s, case):
    hq, g = case["heads"], case["groups"]
    hpg = hq // g
    new, lens = _lens(case)
    out = torch.empty(s["rows"], hq, DH, device=DEV, dtype=torch.float64)
    at = 0
    for b, (n, total) in enumerate(zip(new, lens)):
        ids = s["table"][b][: -(-total // case["page"])].long()
        dead = (torch.arange(total, device=DEV)[None, :]
                > torch.arange(total - n, total, device=DEV)[:, None])
        for h in range(g):
            k = s["k"][ids, h].reshape(-1, DH)[:total].double()
            v = s["v"][ids, h].reshape(-1, DH)[:total].double()
            for i in range(h * hpg, (h + 1) * hpg):
                z = (s["q"][at:at + n, i].double() @ k.T) / math.sqrt(DH)
                out[at:at + n, i] = torch.softmax(z.masked_fill(dead, -math.inf), -1) @ v
        at += n
    return out


def _exact_sample(s, case):
    out = []
    for b in range(case["rows"]):
        x = s["logits"][b].double().cpu()
        t = float(s["temperature"][b])
        if t == 0:
            out.append(int((x == x.max()).nonzero()[0]))
            continue
        w = torch.exp((x - x.max()) / t)
        order = torch.argsort(x, descending=True, stable=True)
        k, p, mp = int(s["top_k"][b]), float(s["top_p"][b]), float(s["min_p"][b])
        if k > 0:
            order = order[:k]
        if p < 1:
            c = torch.cumsum(w[order], 0)
            order = order[: max(1, int((c - w[order] < p * c[-1]).sum()))]
        kept = order[w[order] >= mp]
        order = kept if len(kept) else order[:1]
        ids = torch.sort(order).values
        c = torch.cumsum(w[ids], 0)
        out.append(int(ids[int((c <= float(s["u"][b]) * c[-1]).sum())]))
    return torch.tensor(out, device=DEV)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend,
            "sample": _exact_sample}[case["op"]](s, case)
